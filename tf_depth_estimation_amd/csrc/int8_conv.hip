// Convolutions as products of 8-bit integers with a scale per input pixel (token) and per output channel
// (include/tde.h, "8-bit activations" (1)): row quantiser, weight quantiser, and the conv / transposed conv with
// bias + ReLU.
//
//   y[p, k] = relu?( ws[k] * sum_t xs[p(t)] * (sum_c xq[p(t), c] wq[t, k, c]) + b[k] )
//
// A pixel's scale differs from tap to tap, so the integer sum ends with each tap: it is converted and added into an fp32
// accumulator with its pixel's scale.  The product is taken transposed (weights are the matrix instruction's rows,
// pixels its columns): then a lane's four results are four channels of ONE pixel, so the scale is one register per
// tile, loaded by the lane that needs it, and the result leaves as one 16-byte store.
#include "int8_common.h"
#include "split_math.h"      // FDiv: division by a launch constant

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));

// code bytes of a row of C channels: the reduction depth of one matrix instruction (32 or 64)
inline int q8_row(int C) { return C <= 32 ? 32 : (C + 63) / 64 * 64; }
inline int q8_cols(int K) { return (K + 15) / 16 * 16; }
constexpr int Q8_MAXC = 4096;
constexpr long Q8_MAXPIX = 1 << 26;      // pixels of an input or output: a grid's threads stay below 2^32

// a / 127, correctly rounded: the product with the rounded reciprocal and one step with its exact remainder.  Below 2^-100,
// where the remainder may be no normal number, by way of fp64: a's 24 bits over 127 never come so near the middle between
// two fp32 numbers that the fp64 rounding could pass it (24 + 7 bits of numerator and denominator, 53 of quotient).
__device__ __forceinline__ float q8_scale(unsigned amax_bits) {
  const float a = __uint_as_float(amax_bits);
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  if (a < 0x1p-100f) return (float)((double)a / 127.0);
  const float q = a * (1.f / 127.f);
  return fmaf(fmaf(-q, 127.f, a), 1.f / 127.f, q);
}

// rne(127 x / a), exact.  The fp32 estimate t = x * (127 / a) is off by less than 4e-5 (three roundings of at most 127),
// so unless t lies that close to a half-integer its rounding is the quotient's.  Near one (1 element in 10^4) the quotient
// lies between floor(t) and floor(t) + 1, and the sign of 254 x - (2 floor(t) + 1) a decides (both products are exact in
// fp64: 32 bits), 0 being a tie, to even.  Where 1 / a may be no normal number x and a are first scaled by a power of two (an
// x that this makes subnormal has code 0 anyway).  a: finite maximum, |x| <= a.
struct Q8Div {
  float a, inv, sc;          // inv 0: the row is zero or not finite
};
__device__ __forceinline__ Q8Div q8_div(unsigned amax_bits) {
  Q8Div d;
  d.a = __uint_as_float(amax_bits);
  d.sc = d.a < 0x1p-100f ? 0x1p64f : (d.a > 0x1p100f ? 0x1p-64f : 1.f);
  d.inv = amax_bits == 0 || amax_bits >= 0x7f800000u ? 0.f : 127.f * __builtin_amdgcn_rcpf(d.a * d.sc);
  return d;
}
// codes of four channels, packed.  (1.5 * 2^23 + t is rounded to an integer, whose code is then its low byte.)
__device__ __forceinline__ int q8_code4(const f4& x, const Q8Div& d) {
  constexpr float MAGIC = 0x1.8p23f;
  f4 t = x, r, e;
  if (d.sc != 1.f)
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] *= d.sc;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r[j] = fmaf(t[j], d.inv, MAGIC);
    e[j] = fabsf(fmaf(t[j], d.inv, MAGIC - r[j]));
  }
  // (inv 0: t is 0 or, where x is not finite, NaN; either way the row's codes are 0)
  if (fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])) > 0.49995f)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float k = floorf(t[j] * d.inv);
      const double s = 254.0 * (double)x[j] - (double)(2.f * k + 1.f) * (double)d.a;
      r[j] = MAGIC + (s > 0.0 || (s == 0.0 && ((int)k & 1)) ? k + 1.f : k);
    }
  const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(r[1]), __float_as_uint(r[0]), 0x0c0c0400);
  const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(r[3]), __float_as_uint(r[2]), 0x0c0c0400);
  return d.inv == 0.f ? 0 : (int)__builtin_amdgcn_perm(hi, lo, 0x05040100);
}

// ---- rows: L lanes per row (a power of two <= 64), QPL quads of channels per lane and RT rows held in registers, so that
// a lane has about four loads in flight; VEC: 16-byte loads.  Quantises rows row, row + R, .. (px: this lane's first quad of
// the first, step: elements from one to the next); row `rows` becomes zero.  IN: all of them lie before the last row.
template <int L, int QPL, int RT, bool VEC, bool IN, class Put, class PutScale>
__device__ __forceinline__ void q8_quantize(int l, int row, int R, int rows, int C, int Cp, const float* px, long step,
                                            Put put, PutScale put_scale) {
  f4 v[RT][QPL];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const float* pt = px + t * step;
#pragma unroll
    for (int i = 0; i < QPL; ++i) {
      const int c = 4 * (l + i * L);
      v[t][i] = f4{0.f, 0.f, 0.f, 0.f};
      if ((IN || row + t * R < rows) && c < C) {
        if (VEC && (IN || c + 3 < C || row + t * R + 1 < rows)) {      // (the last row's padding may lie behind the tensor)
          v[t][i] = *reinterpret_cast<const f4*>(pt + 4 * i * L);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + j < C) v[t][i][j] = pt[4 * i * L + j];
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    if (!IN && row + t * R > rows) break;
    unsigned am = 0;
#pragma unroll
    for (int i = 0; i < QPL; ++i) {
      if (VEC && (C & 3))            // a last quad that holds the view's padding
#pragma unroll
        for (int j = 1; j < 4; ++j)
          if (4 * (l + i * L) + j >= C) v[t][i][j] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) am = max(am, abs_bits(v[t][i][j]));
    }
    am = group_umax<L>(am);
    const Q8Div d = q8_div(am);
#pragma unroll
    for (int i = 0; i < QPL; ++i)
      if (4 * (l + i * L) < Cp) put(t, i, 4 * i * L < C ? q8_code4(v[t][i], d) : 0);
    if (l == 0) put_scale(t, q8_scale(am));      // (row `rows`: no channel was read, scale 0)
  }
}
// 196608 x 128 19.5 us (6.5 TB/s of reads and writes), 43200 x 512 18.2 us (6.1), 393216 x 32 11.9 us (5.4; half of it VALU
// work: 20 instructions for four codes, and a row's maximum and scale); few rows 2.4 us, a launch's latency.  Two quads a lane
// share the row's work: 393216 x 32 13.3 us with one, 393216 x 64 19.7 us, 20.9 with one and 22.5 with four.
template <int L, int QPL, int RT, bool VEC>
__global__ void __launch_bounds__(256) q8_rows_kernel(int rows, int C, int Cp, const float* x, long cs, int8_t* codes,
                                                      float* scales) {
  constexpr int R = 256 / L;
  const int l = threadIdx.x % L, g = L == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / L) : threadIdx.x / L;
  const long xo = g * cs + 4 * l;
  const int qo = g * Cp + 4 * l;
  for (int rb = blockIdx.x * (R * RT); rb <= rows; rb += gridDim.x * (R * RT)) {      // (uniform: scalar addresses)
    const float* const px = x + rb * cs + xo;
    const auto put = [&](int t, int i, int q) { *reinterpret_cast<int*>(codes + (long)(rb + t * R) * Cp + 4 * i * L + qo) = q; };
    const auto put_scale = [&](int t, float sc) { (scales + rb + t * R)[g] = sc; };
    if (rb + R * RT < rows) q8_quantize<L, QPL, RT, VEC, true>(l, rb + g, R, rows, C, Cp, px, R * cs, put, put_scale);
    else q8_quantize<L, QPL, RT, VEC, false>(l, rb + g, R, rows, C, Cp, px, R * cs, put, put_scale);
  }
}

// ---- long rows: 256 lanes each, so that few rows are not one wave's work and many keep few registers (8192 x 2048 14.5 us,
// 5.8 TB/s, and 17.4 with a wave per row; one row of 4096 2.8 / 6.0)
template <int QPL, bool VEC>
__global__ void __launch_bounds__(256) q8_rows_wide_kernel(long rows, int C, int Cp, const float* x, long cs, int co,
                                                           int8_t* codes, float* scales) {
  __shared__ unsigned mx[4];
  const long row = (long)blockIdx.y * 65535 + blockIdx.x;
  if (row > rows) return;
  const float* px = x + row * cs + co;
  f4 v[QPL];
  unsigned am = 0;
#pragma unroll
  for (int i = 0; i < QPL; ++i) {
    const int c = 4 * (threadIdx.x + i * 256);
    v[i] = f4{0.f, 0.f, 0.f, 0.f};
    if (row < rows && c < C) {
      if (VEC && c + 3 < C) {
        v[i] = *reinterpret_cast<const f4*>(px + c);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < C) v[i][j] = px[c + j];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < QPL; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) am = max(am, abs_bits(v[i][j]));
  am = group_umax<64>(am);
  if ((threadIdx.x & 63) == 0) mx[threadIdx.x >> 6] = am;
  __syncthreads();
  am = max(max(mx[0], mx[1]), max(mx[2], mx[3]));
  const Q8Div d = q8_div(am);
#pragma unroll
  for (int i = 0; i < QPL; ++i) {
    const int c = 4 * (threadIdx.x + i * 256);
    if (c < Cp) *reinterpret_cast<int*>(codes + row * Cp + c) = q8_code4(v[i], d);
  }
  if (threadIdx.x == 0) scales[row] = q8_scale(am);
}

// ---- weights: a block takes four output channels (padding channels write zeros), 256 lanes each; lanes run along the
// contiguous dimension of the layout (0: output channels, 1: input channels).  The maximum's atomics are on integers in
// LDS: the order does not matter.
__global__ void __launch_bounds__(1024) q8_weights_kernel(int taps, int cin, int K, int Kp, int Cp, int layout,
                                                          const float* w, int8_t* codes, float* scales) {
  constexpr int KB = 4, NL = 1024 / KB;
  __shared__ unsigned mx[KB];
  const int kk = layout == 0 ? threadIdx.x % KB : threadIdx.x / NL, rl = layout == 0 ? threadIdx.x / KB : threadIdx.x % NL;
  const int k = blockIdx.x * KB + kk, rows = taps * cin;
  if (threadIdx.x < KB) mx[threadIdx.x] = 0;
  __syncthreads();
  // element (tap t, input channel c) of this channel; the two layouts' strides
  const long st = layout == 0 ? (long)cin * K : (long)K * cin, sc = layout == 0 ? K : 1;
  const float* wk = w + (layout == 0 ? (long)k : (long)k * cin);
  unsigned am = 0;
  if (k < K) {
#pragma unroll 4
    for (int i = rl; i < rows; i += NL) {
      const int t = i / cin, c = i - t * cin;
      am = max(am, abs_bits(wk[t * st + c * sc]));
    }
    atomicMax(&mx[kk], am);
  }
  __syncthreads();
  am = mx[kk];
  const Q8Div d = q8_div(am);
  const int nq = Cp / 4, quads = taps * nq;
#pragma unroll 2
  for (int i = rl; i < quads; i += NL) {
    const int t = i / nq, c = 4 * (i - t * nq);
    f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k < K && c + j < cin) v[j] = wk[t * st + (c + j) * sc];
    *reinterpret_cast<int*>(codes + ((long)t * Kp + k) * Cp + c) = q8_code4(v, d);
  }
  if (rl == 0) scales[k] = q8_scale(am);
}

// The same for layout 0 with K % 4 == 0 and 16-byte rows: a lane reads four output channels at a time, and writes four
// codes of each from four rows turned in registers.  Block = 16 channels x 256 rows.  (3x3x512 -> 512: 19 us, 31 by the
// kernel above; 2048 x 2048: 15.)
__global__ void __launch_bounds__(1024) q8_weights4_kernel(int taps, int cin, int K, int Kp, int Cp, const float* w,
                                                           int8_t* codes, float* scales) {
  __shared__ unsigned mx[16];
  const int kl = 4 * (threadIdx.x & 3), rl = threadIdx.x >> 2, k = blockIdx.x * 16 + kl, rows = taps * cin;
  const bool on = k < K;
  if (threadIdx.x < 16) mx[threadIdx.x] = 0;
  __syncthreads();
  unsigned am[4] = {0, 0, 0, 0};
  if (on) {
#pragma unroll 6
    for (int i = rl; i < rows; i += 256) {
      const f4 v = *reinterpret_cast<const f4*>(w + (long)i * K + k);
#pragma unroll
      for (int j = 0; j < 4; ++j) am[j] = max(am[j], abs_bits(v[j]));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) atomicMax(&mx[kl + j], am[j]);
  }
  __syncthreads();
  Q8Div d[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) d[j] = q8_div(mx[kl + j]);
  const int nq = Cp / 4, quads = taps * nq;
#pragma unroll 2
  for (int i = rl; i < quads; i += 256) {
    const int t = i / nq, c = 4 * (i - t * nq);
    f4 v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v[r] = f4{0.f, 0.f, 0.f, 0.f};
      if (on && c + r < cin) v[r] = *reinterpret_cast<const f4*>(w + ((long)t * cin + c + r) * K + k);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<int*>(codes + ((long)t * Kp + k + j) * Cp + c) = q8_code4(f4{v[0][j], v[1][j], v[2][j], v[3][j]}, d[j]);
  }
  if (rl == 0)
#pragma unroll
    for (int j = 0; j < 4; ++j) scales[k + j] = q8_scale(mx[kl + j]);
}

// ---- the product.  One class of output pixels (a conv has one; a stride-s transposed conv s * s parities): output
// pixel (i, j) of the class's GH x GW grid lies at (i * os + py, j * os + px) and reads, through tap (ty, tx),
// input pixel (i * is + iy0 + dir * ty, ...) with weights of tap (ky0 + kst * ty, ...).
struct Q8Conv {
  int N, H, W;               // input pixels
  int OH, OW;                // output pixels
  int Cp, K, Kp;             // code bytes of a row, output channels (real, padded)
  int KH, KW, is, os, dir, kst, pt, pl, deconv;
  const int8_t* x;
  const float* xs;
  const int8_t* w;
  const float *ws, *bias;
  float* y;
  int ycs, yco, relu, vec;
};

struct Q8Class {
  int GH, GW, M, py, px, iy0, ix0, ky0, kx0, nty, ntx;
};
__device__ __forceinline__ Q8Class q8_class(const Q8Conv& p, int z) {
  Q8Class c;
  if (!p.deconv) {
    c.GH = p.OH; c.GW = p.OW; c.py = c.px = 0;
    c.iy0 = -p.pt; c.ix0 = -p.pl; c.ky0 = c.kx0 = 0;
    c.nty = p.KH; c.ntx = p.KW;
  } else {
    c.py = z / p.os; c.px = z - c.py * p.os;
    c.GH = (p.OH - c.py + p.os - 1) / p.os; c.GW = (p.OW - c.px + p.os - 1) / p.os;
    c.ky0 = (c.py + p.pt) % p.os; c.kx0 = (c.px + p.pl) % p.os;
    c.iy0 = (c.py + p.pt) / p.os; c.ix0 = (c.px + p.pl) / p.os;
    c.nty = c.ky0 < p.KH ? (p.KH - c.ky0 + p.os - 1) / p.os : 0;
    c.ntx = c.kx0 < p.KW ? (p.KW - c.kx0 + p.os - 1) / p.os : 0;
  }
  c.M = p.N * c.GH * c.GW;
  return c;
}

template <int KC>
struct Q8Frag;
template <>
struct Q8Frag<64> {
  typedef i4 T;
  static __device__ __forceinline__ i4 mfma(T a, T b, i4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};
template <>
struct Q8Frag<32> {
  typedef long T;
  static __device__ __forceinline__ i4 mfma(T a, T b, i4 c) { return __builtin_amdgcn_mfma_i32_16x16x32_i8(a, b, c, 0, 0, 0); }
};

// scales and biases of a lane's channels (k0 + 16 a ..+3), loaded together before the stores
template <int TM>
struct Q8Epi {
  f4 ws[TM], bs[TM];
  __device__ __forceinline__ Q8Epi(const Q8Conv& p, int k0) {
#pragma unroll
    for (int a = 0; a < TM; ++a) {
      const int k = k0 + 16 * a;
      ws[a] = bs[a] = f4{0.f, 0.f, 0.f, 0.f};
      if (k < p.K) {
        ws[a] = *reinterpret_cast<const f4*>(p.ws + k);       // (scales are padded to Kp)
        if (p.bias)
#pragma unroll
          for (int e = 0; e < 4; ++e) bs[a][e] = p.bias[min(k + e, p.K - 1)];
      }
    }
  }
  // scale, bias, ReLU and store of tile a: four channels of the pixel at py
  __device__ __forceinline__ void store(const Q8Conv& p, float* py, int k0, int a, const f4& acc) const {
    const int k = k0 + 16 * a;
    if (k >= p.K) return;
    f4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = fmaf(acc[e], ws[a][e], bs[a][e]);
      o[e] = p.relu && v < 0.f ? 0.f : v;
    }
    if (p.vec && k + 3 < p.K) {
      tde_st(reinterpret_cast<f4*>(py + k), o);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k + e < p.K) py[k + e] = o[e];
    }
  }
};
__device__ __forceinline__ float* q8_out(const Q8Conv& p, const Q8Class& cl, int n, int i, int j) {
  return p.y + (((long)n * p.OH + i * p.os + cl.py) * p.OW + j * p.os + cl.px) * p.ycs + p.yco;
}

// ---- few pixels: WK waves take turns at the (tap, channel chunk) steps of a tile of 16 TM channels x 16 TN pixels and
// add their fp32 sums through LDS in wave order.  The time is the latency of the weights, which come straight from the
// caches (a lane's 16 / 8 bytes are its row's k-quarter); the waves of a SIMD cover it for each other.  (4x4x512 -> 512, one
// image: 6.6 us; with the fragments of 2 / 4 steps in flight per wave 7.0 / 7.8: their addresses delay the first load.)
template <int TM, int TN, int KC, int WK>
__global__ void __launch_bounds__(64 * WK) q8_split_kernel(const Q8Conv p) {
  using F = typename Q8Frag<KC>::T;
  __shared__ f4 red[(WK - 1) * TM * TN * 64];
  const int lane = threadIdx.x & 63, wk = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, kq = lane >> 4;
  const Q8Class cl = q8_class(p, blockIdx.z);
  const int m0 = blockIdx.x * 16 * TN, n0 = blockIdx.y * 16 * TM;
  const long zero_row = (long)p.N * p.H * p.W;

  int iy[TN], ix[TN];
  long pb[TN];
#pragma unroll
  for (int b = 0; b < TN; ++b) {
    const int m = m0 + 16 * b + r16;
    if (m < cl.M) {
      const int hw = cl.GH * cl.GW, n = m / hw, r = m - n * hw, i = r / cl.GW, j = r - i * cl.GW;
      iy[b] = i * p.is + cl.iy0; ix[b] = j * p.is + cl.ix0;
      pb[b] = (long)n * p.H * p.W;
    } else {
      iy[b] = -(1 << 29); ix[b] = 0; pb[b] = 0;      // no tap reaches the image: the zero row
    }
  }
  const int8_t* wrow[TM];
#pragma unroll
  for (int a = 0; a < TM; ++a) wrow[a] = p.w + (long)min(n0 + 16 * a + r16, p.Kp - 1) * p.Cp + kq * (KC / 4);

  f4 acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b) acc[a][b] = f4{0.f, 0.f, 0.f, 0.f};

  const int nch = p.Cp / KC, steps = cl.nty * cl.ntx * nch;
  for (int s = wk; s < steps; s += WK) {
    const int t = s / nch, ch = s - t * nch, ty = t / cl.ntx, tx = t - ty * cl.ntx;
    const long wtap = ((long)(cl.ky0 + p.kst * ty) * p.KW + cl.kx0 + p.kst * tx) * p.Kp * p.Cp + ch * KC;
    F fa[TM], fb[TN];
    float xs[TN];
#pragma unroll
    for (int a = 0; a < TM; ++a) fa[a] = *reinterpret_cast<const F*>(wrow[a] + wtap);
#pragma unroll
    for (int b = 0; b < TN; ++b) {
      const int yy = iy[b] + p.dir * ty, xx = ix[b] + p.dir * tx;
      const bool in = (unsigned)yy < (unsigned)p.H && (unsigned)xx < (unsigned)p.W;
      const long pix = in ? pb[b] + (long)yy * p.W + xx : zero_row;
      fb[b] = *reinterpret_cast<const F*>(p.x + pix * p.Cp + kq * (KC / 4) + ch * KC);
      xs[b] = p.xs[pix];
    }
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b) {
        const i4 ia = Q8Frag<KC>::mfma(fa[a], fb[b], i4{0, 0, 0, 0});
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[a][b][j] = fmaf((float)ia[j], xs[b], acc[a][b][j]);
      }
  }

  if (wk > 0)
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b) red[((wk - 1) * TM * TN + a * TN + b) * 64 + lane] = acc[a][b];
  __syncthreads();
  if (wk > 0) return;
  for (int w = 0; w < WK - 1; ++w)
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b) acc[a][b] += red[(w * TM * TN + a * TN + b) * 64 + lane];
  const Q8Epi<TM> epi(p, n0 + 4 * kq);
#pragma unroll
  for (int b = 0; b < TN; ++b) {
    const int m = m0 + 16 * b + r16;
    if (m >= cl.M) continue;
    const int hw = cl.GH * cl.GW, n = m / hw, r = m - n * hw, i = r / cl.GW, j = r - i * cl.GW;
    float* py = q8_out(p, cl, n, i, j);
#pragma unroll
    for (int a = 0; a < TM; ++a) epi.store(p, py, n0 + 4 * kq, a, acc[a][b]);
  }
}

// ---- the same on the fp32 input, in one launch: a block of 16 channels x 16 pixels quantises the input pixels that its
// taps reach into LDS by itself (rows [scale | codes] as in the kernel below), the weights of its first U steps in flight
// meanwhile.  Each of the ceil(K / 16) blocks of the same pixels does that work again, so this serves where it is small (up to
// 32 rows) and a launch counts.  4x4x512 -> 512 9.5 us in a graph, as the two kernels (9.2), but 9.4 / 13.7 called one after
// the other, where the host's launches are the time; one token of 1024 -> 1024 channels 5.4 / 6.6.
struct Q8Src {
  const float* x;            // channel view of the input
  long cs;
  int C, cap;                // channels, LDS rows of pixels
};
template <int QPL, int RT>
__global__ void __launch_bounds__(1024) q8_small_kernel(const Q8Conv p, const Q8Src in) {
  constexpr int WK = 16, KC = 64, HEAD = 16, U = 4;
  extern __shared__ __attribute__((aligned(16))) char q8_lds[];
  const int lane = threadIdx.x & 63, wk = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, kq = lane >> 4;
  const Q8Class cl = q8_class(p, blockIdx.z);
  const int m0 = blockIdx.x * 16, n0 = blockIdx.y * 16;
  if (m0 >= cl.M) return;                                   // (pixels are counted for the largest class)
  const int RB = p.Cp + HEAD;

  const int nch = p.Cp / KC, steps = cl.nty * cl.ntx * nch;
  const int8_t* const wrow = p.w + (long)(n0 + r16) * p.Cp + kq * (KC / 4);
  auto wload = [&](int s) __attribute__((always_inline)) {
    const int t = s / nch, ch = s - t * nch, ty = t / cl.ntx, tx = t - ty * cl.ntx;
    return *reinterpret_cast<const i4*>(wrow + ((long)(cl.ky0 + p.kst * ty) * p.KW + cl.kx0 + p.kst * tx) * p.Kp * p.Cp +
                                        ch * KC);
  };
  i4 fa[U];
#pragma unroll
  for (int u = 0; u < U; ++u) fa[u] = wk + u * WK < steps ? wload(wk + u * WK) : i4{0, 0, 0, 0};

  // the input pixels [base, base + rows) that the block's taps reach: whole images, rows of one, or part of a row
  const int hw = cl.GH * cl.GW, HW = p.H * p.W, mh = min(m0 + 15, cl.M - 1);
  const int nl = m0 / hw, nh = mh / hw;
  long base = (long)nl * HW;
  int rows = (nh - nl + 1) * HW;
  if (nl == nh) {
    const int rl = m0 - nl * hw, rh = mh - nh * hw, il = rl / cl.GW, ih = rh / cl.GW;
    const int yb = p.dir < 0 ? cl.nty - 1 : 0, yf = p.dir < 0 ? 0 : cl.nty - 1;
    const int yl = max(il * p.is + cl.iy0 - yb, 0), yh = min(ih * p.is + cl.iy0 + yf, p.H - 1);
    int xl = 0, xh = p.W - 1;
    if (il == ih) {
      const int xb = p.dir < 0 ? cl.ntx - 1 : 0, xf = p.dir < 0 ? 0 : cl.ntx - 1;
      xl = max((rl - il * cl.GW) * p.is + cl.ix0 - xb, 0);
      xh = min((rh - ih * cl.GW) * p.is + cl.ix0 + xf, p.W - 1);
    }
    base += (long)yl * p.W + xl;
    rows = max((yh - yl) * p.W + xh - xl + 1, 0);           // (0: no tap reaches the image)
  }
  rows = min(rows, in.cap);
  for (int r0 = wk; r0 <= rows; r0 += WK * RT)
    q8_quantize<64, QPL, RT, true, false>(
        lane, r0, WK, rows, in.C, p.Cp, in.x + (base + r0) * in.cs + 4 * lane, WK * in.cs,
        [&](int t, int i, int q) {
          *reinterpret_cast<int*>(q8_lds + (r0 + t * WK) * RB + HEAD + 4 * (lane + 64 * i)) = q;
        },
        [&](int t, float sc) { *reinterpret_cast<float*>(q8_lds + (r0 + t * WK) * RB) = sc; });
  __syncthreads();

  const int m = m0 + r16, n = m / hw, rr = m - n * hw, i = rr / cl.GW, j = rr - i * cl.GW;
  const int iy = m < cl.M ? i * p.is + cl.iy0 : -(1 << 29), ix = j * p.is + cl.ix0;
  const int pb = (int)((long)n * HW - base);
  f4 acc = {0.f, 0.f, 0.f, 0.f};
  auto step = [&](int s, const i4& a) __attribute__((always_inline)) {
    const int t = s / nch, ch = s - t * nch, ty = t / cl.ntx, tx = t - ty * cl.ntx;
    const int yy = iy + p.dir * ty, xx = ix + p.dir * tx;
    const bool inside = (unsigned)yy < (unsigned)p.H && (unsigned)xx < (unsigned)p.W;
    const char* row = q8_lds + (inside ? pb + yy * p.W + xx : rows) * RB;
    const i4 ia = Q8Frag<KC>::mfma(a, *reinterpret_cast<const i4*>(row + HEAD + kq * (KC / 4) + ch * KC), i4{0, 0, 0, 0});
    const float xs = *reinterpret_cast<const float*>(row);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf((float)ia[e], xs, acc[e]);
  };
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (wk + u * WK < steps) step(wk + u * WK, fa[u]);
  for (int s = wk + U * WK; s < steps; s += WK) step(s, wload(s));

  f4* red = reinterpret_cast<f4*>(q8_lds + (in.cap + 1) * RB);
  if (wk > 0) red[(wk - 1) * 64 + lane] = acc;
  __syncthreads();
  if (wk > 0) return;
#pragma unroll
  for (int w = 0; w < WK - 1; ++w) acc += red[w * 64 + lane];
  const Q8Epi<1> epi(p, n0 + 4 * kq);
  if (m < cl.M) epi.store(p, q8_out(p, cl, n, i, j), n0 + 4 * kq, 0, acc);
}

// ---- maps: a block computes 16 TM WC channels of a TH x TW tile of pixels (16 TN WP of them) of one image and class.  The
// input pixels its taps reach lie in LDS as a patch of rows [scale | codes] (`cb` bytes of channels at a time), zero
// outside the image, so a tap is one uniform offset into it and needs no address or bounds arithmetic; the weights come
// from the caches, two steps (tap, channel chunk) ahead.  The scale's 16 (8) bytes also pad the rows, so that the
// fragments of 8 (16) neighbouring pixels lie in different banks.  WK groups of waves split the steps where there are few
// tiles, and add their sums through LDS in order.  ONE: a tap is one step (the usual case of few channels), no loop.
// What bounds it there: a tap's conversion is 8 VALU instructions per 16x16 tile, 32 cycles, against 16 (8) cycles of the
// matrix unit (96x128x32 -> 32, 7x7, batch 32: 68 us = 580 TOP/s, the VALU busy 91 %, the matrix unit 28 %).  (The second
// launch bound keeps the products out of the accumulator file: with it, 2 moves per result and step cost more than the
// products.)
struct Q8Tile {
  int lw, tx, ty, cb;        // log2 of the tile width, tiles per row and column of the class grid, channel bytes per patch fill
  int PH, PW;                // patch rows and columns (of the class with the most taps)
  FDiv fPW, fnq, fnq1;       // by PW, by the 16-byte pieces of a pixel in a fill and in the last one
};

template <int TM, int TN, int KC, bool ONE, int WC, int WP, int WK>
__global__ void __launch_bounds__(64 * WC * WP * WK, 2) q8_halo_kernel(const Q8Conv p, const Q8Tile tl) {
  using F = typename Q8Frag<KC>::T;
  constexpr int NT = 64 * WC * WP * WK, BP = 16 * TN * WP, HEAD = KC / 4;
  extern __shared__ __attribute__((aligned(16))) char q8_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wc = wv % WC, wp = wv / WC % WP, wk = wv / (WC * WP);
  const int r16 = lane & 15, kq = lane >> 4;
  const Q8Class cl = q8_class(p, blockIdx.z);
  const int per = tl.tx * tl.ty;
  const int n = blockIdx.x / per, rem = blockIdx.x - n * per, tyi = rem / tl.tx, txi = rem - tyi * tl.tx;
  const int TW = 1 << tl.lw, i0 = tyi * (BP >> tl.lw), j0 = txi * TW;
  if (i0 >= cl.GH || j0 >= cl.GW) return;                   // (tiles are counted for the largest class)
  const int n0 = (blockIdx.y * WC + wc) * 16 * TM;
  const int PW = tl.PW, NP = tl.PH * PW;
  const int back = p.dir < 0;
  const int oy = i0 * p.is + cl.iy0 - (back ? cl.nty - 1 : 0), ox = j0 * p.is + cl.ix0 - (back ? cl.ntx - 1 : 0);
  const int RB = tl.cb + HEAD;                              // bytes of a patch row

  int prow[TN];                                             // this lane's pixels in the patch (bytes), at tap offset 0
#pragma unroll
  for (int b = 0; b < TN; ++b) {
    const int q = 16 * (wp * TN + b) + r16, i = q >> tl.lw, j = q & (TW - 1);
    prow[b] = (i * PW + j) * p.is * RB;
  }
  const int kofs = HEAD + kq * (KC / 4);                    // this lane's k-quarter in a row
  unsigned wrow[TM];                                        // ... and its weight rows in a tap's plane
#pragma unroll
  for (int a = 0; a < TM; ++a) wrow[a] = (unsigned)min(n0 + 16 * a + r16, p.Kp - 1) * (unsigned)p.Cp + kq * (KC / 4);
  const int dy = (back ? -PW : PW) * RB, dx = back ? -RB : RB;
  const int org = back ? ((cl.nty - 1) * PW + cl.ntx - 1) * RB : 0;      // patch offset of tap (0, 0)

  f4 acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b) acc[a][b] = f4{0.f, 0.f, 0.f, 0.f};

  const int taps = cl.nty * cl.ntx;
  for (int c0 = 0; c0 < p.Cp && taps > 0; c0 += tl.cb) {
    const int cbytes = min(tl.cb, p.Cp - c0), nq = cbytes / 16, total = NP * nq;
    if (c0 > 0) __syncthreads();                            // the last fill's fragments have been read
    const FDiv fnq = c0 + tl.cb < p.Cp ? tl.fnq : tl.fnq1;
    constexpr int U = 4;                                    // pieces in flight per lane (8: 169 registers, two waves a SIMD)
    for (int base = tid; base < total; base += U * NT) {
      i4 v[U];
      int dst[U];
      float sc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int idx = base + u * NT;
        v[u] = i4{0, 0, 0, 0};
        sc[u] = -1.f;                                       // (a scale is never negative: not a row's first piece)
        dst[u] = -1;
        if (idx < total) {
          const int pp = fdiv(idx, fnq), c = idx - pp * nq, y = fdiv(pp, tl.fPW), x = pp - y * PW, iy = oy + y, ix = ox + x;
          dst[u] = pp * RB + HEAD + 16 * c;
          if (c == 0) sc[u] = 0.f;
          if ((unsigned)iy < (unsigned)p.H && (unsigned)ix < (unsigned)p.W) {
            const long pix = ((long)n * p.H + iy) * p.W + ix;
            v[u] = *reinterpret_cast<const i4*>(p.x + pix * p.Cp + c0 + 16 * c);
            if (c == 0) sc[u] = p.xs[pix];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (dst[u] >= 0) {
          if (KC == 64) {
            *reinterpret_cast<i4*>(q8_lds + dst[u]) = v[u];
          } else {                                          // (rows of 40 bytes: 8-byte aligned)
            int2* d = reinterpret_cast<int2*>(q8_lds + dst[u]);
            d[0] = int2{v[u][0], v[u][1]};
            d[1] = int2{v[u][2], v[u][3]};
          }
          if (!(sc[u] < 0.f)) *reinterpret_cast<float*>(q8_lds + dst[u] - HEAD) = sc[u];
        }
    }
    __syncthreads();

    // this wave group's steps, the weights of the next two in flight
    const int nch = ONE ? 1 : cbytes / KC, steps = taps * nch;
    const int s0 = steps * wk / WK, s1 = steps * (wk + 1) / WK;
    if (s0 < s1) {
      const int t0 = s0 / nch, ch0 = s0 - t0 * nch, ty0 = t0 / cl.ntx, tx0 = t0 - ty0 * cl.ntx;
      int lch = ch0, lty = ty0, ltx = tx0;                  // step to load
      int ch = ch0, ty = ty0, tx = tx0, s = s0;             // step to compute
      const long plane = (long)p.Kp * p.Cp;
      const long wx = p.kst * plane, wy = p.kst * p.KW * plane - (cl.ntx - 1) * wx;      // to the next tap, the next row
      const int8_t* const w0 = p.w + ((long)cl.ky0 * p.KW + cl.kx0) * plane + c0;
      const int8_t* wt = w0 + ((long)p.kst * ty0 * p.KW + p.kst * tx0) * plane;
      auto load = [&](F(&f)[TM]) __attribute__((always_inline)) {
        const int8_t* wl = ONE ? wt : wt + lch * KC;
#pragma unroll
        for (int a = 0; a < TM; ++a) f[a] = *reinterpret_cast<const F*>(wl + wrow[a]);
        const bool nt = ONE || lch + 1 == nch, nr = nt && ltx + 1 == cl.ntx, end = nr && lty + 1 == cl.nty;
        lch = nt ? 0 : lch + 1;
        ltx = nr ? 0 : (nt ? ltx + 1 : ltx);
        lty = end ? 0 : (nr ? lty + 1 : lty);               // (past the last step: the first tap again)
        wt = end ? w0 : wt + (nr ? wy : (nt ? wx : 0));
      };
      i4 ia[TM][TN];
      if (!ONE)
#pragma unroll
        for (int a = 0; a < TM; ++a)
#pragma unroll
          for (int b = 0; b < TN; ++b) ia[a][b] = i4{0, 0, 0, 0};
      auto step = [&](F(&f)[TM], F(&fl)[TM]) __attribute__((always_inline)) {
        load(fl);
        const char* pt = q8_lds + (org + ty * dy + tx * dx);
        F fb[TN];
        float xs[TN];
#pragma unroll
        for (int b = 0; b < TN; ++b) fb[b] = *reinterpret_cast<const F*>(pt + prow[b] + kofs + (ONE ? 0 : ch * KC));
        if (ONE) {
#pragma unroll
          for (int b = 0; b < TN; ++b) xs[b] = *reinterpret_cast<const float*>(pt + prow[b]);
#pragma unroll
          for (int a = 0; a < TM; ++a)
#pragma unroll
            for (int b = 0; b < TN; ++b) ia[a][b] = Q8Frag<KC>::mfma(f[a], fb[b], i4{0, 0, 0, 0});
        } else {
#pragma unroll
          for (int a = 0; a < TM; ++a)
#pragma unroll
            for (int b = 0; b < TN; ++b) ia[a][b] = Q8Frag<KC>::mfma(f[a], fb[b], ia[a][b]);
        }
        ++s;
        if (ONE || ch + 1 == nch || s == s1) {
          if (!ONE)
#pragma unroll
            for (int b = 0; b < TN; ++b) xs[b] = *reinterpret_cast<const float*>(pt + prow[b]);
#pragma unroll
          for (int a = 0; a < TM; ++a)
#pragma unroll
            for (int b = 0; b < TN; ++b) {
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[a][b][j] = fmaf((float)ia[a][b][j], xs[b], acc[a][b][j]);
              if (!ONE) ia[a][b] = i4{0, 0, 0, 0};
            }
        }
        const bool nt = ONE || ch + 1 == nch, nr = nt && tx + 1 == cl.ntx;
        ch = nt ? 0 : ch + 1;
        tx = nr ? 0 : (nt ? tx + 1 : tx);
        ty = nr ? ty + 1 : ty;
      };
      F f0[TM], f1[TM], f2[TM];
      load(f0);
      load(f1);
      while (true) {
        step(f0, f2);
        if (s == s1) break;
        step(f1, f0);
        if (s == s1) break;
        step(f2, f1);
        if (s == s1) break;
      }
    }
  }

  if (WK > 1) {
    __syncthreads();                                        // the patch has been read: its LDS takes the partial sums
    f4* red = reinterpret_cast<f4*>(q8_lds) + (wp * WC + wc) * (WK - 1) * TM * TN * 64;
    if (wk > 0)
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) red[((wk - 1) * TM * TN + a * TN + b) * 64 + lane] = acc[a][b];
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int w = 0; w < WK - 1; ++w)
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) acc[a][b] += red[(w * TM * TN + a * TN + b) * 64 + lane];
  }
  const Q8Epi<TM> epi(p, n0 + 4 * kq);
#pragma unroll
  for (int b = 0; b < TN; ++b) {
    const int q = 16 * (wp * TN + b) + r16, i = i0 + (q >> tl.lw), j = j0 + (q & (TW - 1));
    if (i >= cl.GH || j >= cl.GW) continue;
    float* py = q8_out(p, cl, n, i, j);
#pragma unroll
    for (int a = 0; a < TM; ++a) epi.store(p, py, n0 + 4 * kq, a, acc[a][b]);
  }
}

// ---- one tap, stride 1: the plain product of M tokens and K weight rows.  Both operands reach LDS by DMA
// (global_load_lds_dwordx4: a wave instruction copies 16 rows of 64 bytes) into a ring of three slots, two steps in
// flight across the barriers; the 16-byte quarters of a row are exchanged by (row >> 1) & 3 on the way, so that the
// fragment reads of 8 neighbouring rows hit different banks.  All sums stay integers until the end.
// 8192 x 2048 x 2048: 42-43 us = 1600-1640 TOP/s with 256 x 256 tiles on 8 waves, whose LDS reads (96 bytes a clock) run
// under the products because the pixel fragments, which every product needs, are read first (55 us the other way round).
// The matrix unit is busy 42 % of the time; the rest are the barriers of a step and the 67 MB that all blocks write at their ends.
// Smaller tiles read more LDS bytes per product and serve where the large ones would leave CUs idle.
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef __attribute__((address_space(1))) void* gbl_ptr_t;
// this wave's LDS reads are done (written as a builtin, so that the compiler knows and waits for none of them again), then
// the barrier
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
template <int N>
__device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <int TM, int TN, int WC, int WP>
__global__ void __launch_bounds__(64 * WC * WP) q8_gemm_kernel(const Q8Conv p, int M, int nct) {
  constexpr int NW = WC * WP, BC = 16 * TM * WC, BP = 16 * TN * WP, NI = (BC + BP) / 16, DI = NI / NW;
  static_assert(NI % NW == 0, "whole DMA instructions per wave");
  constexpr int SLOT = (BC + BP) * 64;
  extern __shared__ __attribute__((aligned(16))) char q8_lds[];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, wc = wv % WC, wp = wv / WC;
  const int r16 = lane & 15, kq = lane >> 4;
  const int lb = tde_xcd_block(blockIdx.x, gridDim.x), pt = lb / nct, ct = lb - pt * nct;
  const int m0 = pt * BP, n0 = ct * BC;

  const int8_t* src[DI];
#pragma unroll
  for (int j = 0; j < DI; ++j) {
    const int row = (wv * DI + j) * 16 + (lane >> 2);
    const int q = ((lane & 3) ^ ((row >> 1) & 3)) * 16;
    const bool in = q < p.Cp;               // rows of 32 bytes: the pixels' upper half is the zero row (row M of the codes)
    src[j] = row < BC ? p.w + (long)min(n0 + row, p.Kp - 1) * p.Cp + (in ? q : q - 32)
                      : p.x + (long)(in ? min(m0 + row - BC, M) : M) * p.Cp + (in ? q : q - 32);
  }
  auto dma = [&](int s, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < DI; ++j)
      __builtin_amdgcn_global_load_lds((gbl_ptr_t)(src[j] + s * 64),
                                       (lds_ptr_t)(q8_lds + slot * SLOT + (wv * DI + j) * 1024), 16, 0, 0);
  };
  i4 acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b) acc[a][b] = i4{0, 0, 0, 0};

  const int lofs = r16 * 64 + ((kq ^ ((r16 >> 1) & 3)) << 4);
  const int steps = (p.Cp + 63) / 64, last = steps - 1;
  struct Frag {
    i4 a[TM], b[TN];
  };
  auto read = [&](Frag& f, int slot) __attribute__((always_inline)) {
    const char* base = q8_lds + slot * SLOT + lofs;
#pragma unroll
    for (int b = 0; b < TN; ++b) f.b[b] = *reinterpret_cast<const i4*>(base + BC * 64 + (wp * TN + b) * 1024);
#pragma unroll
    for (int a = 0; a < TM; ++a) f.a[a] = *reinterpret_cast<const i4*>(base + (wc * TM + a) * 1024);
  };
  auto next = [](int slot) __attribute__((always_inline)) { return slot == 2 ? 0 : slot + 1; };
  // step s: its fragments are in registers; those of step s + 1 are read under its products, step s + 3 replaces it in LDS
  auto step = [&](int s, int slot, const Frag& f, Frag& fn) __attribute__((always_inline)) {
    vm_wait<DI>();        // this wave's part of step s + 1 has landed (step s + 2 may still fly)
    lds_barrier();        // everybody's has, and everybody has read step s
    dma(min(s + 3, last), slot);
    read(fn, next(slot));
    __builtin_amdgcn_sched_barrier(0);      // (left alone, the scheduler puts the reads behind the products)
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b) acc[a][b] = Q8Frag<64>::mfma(f.a[a], f.b[b], acc[a][b]);
  };
  dma(0, 0);
  dma(min(1, last), 1);
  dma(min(2, last), 2);
  Frag f0, f1;
  vm_wait<2 * DI>();
  lds_barrier();
  read(f0, 0);
  int slot = 0;
  for (int s = 0; s < steps; s += 2) {
    step(s, slot, f0, f1);
    slot = next(slot);
    if (s + 1 < steps) step(s + 1, slot, f1, f0);
    slot = next(slot);
  }
  vm_wait<0>();           // no DMA may outlive the block's LDS

  const int k0 = n0 + wc * TM * 16 + 4 * kq;
  const Q8Epi<TM> epi(p, k0);
  float xs[TN];
#pragma unroll
  for (int b = 0; b < TN; ++b) xs[b] = p.xs[min(m0 + (wp * TN + b) * 16 + r16, M)];
#pragma unroll
  for (int b = 0; b < TN; ++b) {
    const int m = m0 + (wp * TN + b) * 16 + r16;
    if (m >= M) continue;
    float* py = p.y + (long)m * p.ycs + p.yco;
#pragma unroll
    for (int a = 0; a < TM; ++a) {
      f4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (float)acc[a][b][j] * xs[b];
      epi.store(p, py, k0, a, v);
    }
  }
}

// ---- launches
template <int TM, int TN, int WK>
void q8_split_launch(const Q8Conv& p, long Mmax, int classes, hipStream_t st) {
  const dim3 grid(tde_cdiv(Mmax, 16 * TN), tde_cdiv(p.K, 16 * TM), classes);
  if (p.Cp % 64 == 0)
    hipLaunchKernelGGL((q8_split_kernel<TM, TN, 64, WK>), grid, dim3(64 * WK), 0, st, p);
  else
    hipLaunchKernelGGL((q8_split_kernel<TM, TN, 32, WK>), grid, dim3(64 * WK), 0, st, p);
}

constexpr int Q8_LDS = 64 * 1024;      // patch bytes of a halo block: two blocks fit a CU's 160 KB

template <int TM, int TN, int WC, int WP, int WK>
bool q8_halo_launch(const Q8Conv& p, int GH, int GW, int classes, hipStream_t st) {
  constexpr int BP = 16 * TN * WP, BC = 16 * TM * WC, NT = 64 * WC * WP * WK;
  constexpr int RED = (WK - 1) * WC * WP * TM * TN * 1024;
  static_assert(RED <= Q8_LDS, "partial sums fit the patch's LDS");
  Q8Tile t;
  t.lw = GW > 8 ? 4 : (GW > 4 ? 3 : 2);
  const int TW = 1 << t.lw, TH = BP / TW, kc = p.Cp % 64 == 0 ? 64 : 32;
  t.PH = (TH - 1) * p.is + (p.KH + p.kst - 1) / p.kst;
  t.PW = (TW - 1) * p.is + (p.KW + p.kst - 1) / p.kst;
  const long NP = (long)t.PH * t.PW;
  t.tx = tde_cdiv(GW, TW); t.ty = tde_cdiv(GH, TH);
  t.cb = (int)(Q8_LDS / NP) - kc / 4;
  t.cb = t.cb >= p.Cp ? p.Cp : t.cb / kc * kc;
  if (t.cb < kc) return false;
  t.fPW = make_fdiv(t.PW);
  t.fnq = make_fdiv(t.cb / 16);
  t.fnq1 = make_fdiv((p.Cp - (p.Cp - 1) / t.cb * t.cb) / 16);
  const int patch = (int)NP * (t.cb + kc / 4), lds = patch > RED ? patch : RED;
  const long blocks = (long)p.N * t.tx * t.ty;
  if (blocks * NT >= (1L << 32)) return false;
  const dim3 grid((unsigned)blocks, tde_cdiv(p.K, BC), classes);
  if (kc == 32)
    hipLaunchKernelGGL((q8_halo_kernel<TM, TN, 32, true, WC, WP, WK>), grid, dim3(NT), lds, st, p, t);
  else if (p.Cp == 64)
    hipLaunchKernelGGL((q8_halo_kernel<TM, TN, 64, true, WC, WP, WK>), grid, dim3(NT), lds, st, p, t);
  else
    hipLaunchKernelGGL((q8_halo_kernel<TM, TN, 64, false, WC, WP, WK>), grid, dim3(NT), lds, st, p, t);
  return true;
}

template <int TM, int TN, int WC, int WP>
void q8_gemm_launch(const Q8Conv& p, int M, hipStream_t st) {
  constexpr int BP = 16 * TN * WP, BC = 16 * TM * WC, LDS = 3 * (BC + BP) * 64;
  if (LDS > 64 * 1024)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&q8_gemm_kernel<TM, TN, WC, WP>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  const int nct = tde_cdiv(p.K, BC);
  hipLaunchKernelGGL((q8_gemm_kernel<TM, TN, WC, WP>), dim3((unsigned)((long)tde_cdiv(M, BP) * nct)), dim3(64 * WC * WP),
                     LDS, st, p, M, nct);
}

int q8_conv(Q8Conv p, hipStream_t st) {
  const int s = p.deconv ? p.os : 1, classes = s * s;
  const int GH = (p.OH + s - 1) / s, GW = (p.OW + s - 1) / s;
  const long Mmax = (long)p.N * GH * GW;
  const long tiles = ((Mmax + 15) / 16) * ((p.K + 15) / 16) * classes;      // 16 x 16 tiles
  if (p.KH == 1 && p.KW == 1 && p.is == 1 && p.os == 1 && p.OH == p.H && p.OW == p.W && (Mmax > 16 || p.Cp < 2048)) {
    // The largest tiles that still fill the CUs.  us, this choice / its neighbour (tokens x input x output channels):
    // 128x2048x2048 5.1 / 6.7 with the next larger tiles, 256x2048x2048 6.9 / 8.8 with the next smaller;
    // 8192x256x256 4.9 / 6.3 (larger), 8192x1024x1024 21.9 / 23.7 (smaller); 393216x64x128 42 / 69 (larger),
    // 49152x512x256 20.9 / 22.6 (smaller).  One token of 2048 -> 2048 channels: 4.2 by the split kernel below, 4.7 here.
    const auto blocks = [&](int k, int m) { return (long)tde_cdiv(Mmax, m) * tde_cdiv(p.K, k); };
    if (blocks(32, 32) <= 256) q8_gemm_launch<1, 1, 2, 2>(p, (int)Mmax, st);
    else if (blocks(64, 64) <= 512) q8_gemm_launch<1, 2, 4, 2>(p, (int)Mmax, st);
    else if (p.K <= 128 || blocks(256, 256) < 192) q8_gemm_launch<2, 4, 2, 2>(p, (int)Mmax, st);
    else q8_gemm_launch<8, 4, 2, 4>(p, (int)Mmax, st);
    return tde_launch_status();
  }
  bool done = false;
  if (GH * GW >= 12 && tiles > 256) {
    // Blocks of fewer pixels and channels, and more wave groups that split the steps, the fewer tiles there are; timed for
    // each size on the networks' layers at batch 1, 8 and 32 (us, this choice / the next larger block):
    // 28x28x256 -> 128 6.3 / 7.9 (14x14x512 -> 256, 208 tiles: 7.9, 7.2 by the split kernel below), 6x8x1024 -> 512 (8)
    // 16.1 / 19.3, 24x32x128 -> 128 (8) 9.3 / 10.3, 24x32x256 -> 128 (8) 11.9 / 13.7, 12x16x512 -> 256 (8) 12.7 / 20.8 (each
    // 10 % and more above that with two waves' channels in one wave), 48x64x64 -> 64 k5 (8) 11.6 / 13.4,
    // 96x128x32 -> 32 k7 (8) 22.0 / 28.2, (32) 64.8 / 72.9 with this choice's smaller neighbour, 24x32x256 -> 128 (32)
    // 23.7 / 28.1
    if (tiles < 512) done = q8_halo_launch<1, 2, 1, 1, 8>(p, GH, GW, classes, st);
    else if (tiles < 1536) done = q8_halo_launch<2, 2, 1, 1, 8>(p, GH, GW, classes, st);
    else if (p.K <= 16) done = tiles < 8192 ? q8_halo_launch<1, 4, 1, 2, 2>(p, GH, GW, classes, st)
                                            : q8_halo_launch<1, 4, 1, 4, 1>(p, GH, GW, classes, st);
    else if (tiles < 4096) done = p.K > 64 ? q8_halo_launch<1, 4, 2, 1, 4>(p, GH, GW, classes, st)
                                           : q8_halo_launch<2, 2, 1, 1, 4>(p, GH, GW, classes, st);
    else if (p.K > 64) done = q8_halo_launch<2, 4, 2, 1, 2>(p, GH, GW, classes, st);
    else if (tiles < 8192) done = q8_halo_launch<2, 2, 1, 2, 2>(p, GH, GW, classes, st);
    else if (p.K > 32) done = q8_halo_launch<2, 4, 2, 2, 1>(p, GH, GW, classes, st);
    else if (tiles < 16384) done = q8_halo_launch<2, 4, 1, 2, 2>(p, GH, GW, classes, st);
    else done = q8_halo_launch<2, 4, 1, 4, 1>(p, GH, GW, classes, st);
  }
  if (!done) {
    // 8x 3x3x512 -> 512 7.0 / 9.3 with the next larger tiles, 16x 9.4 / 11.6 (smaller), 64x 20.2 / 28.0 (smaller)
    if (tiles <= 256) q8_split_launch<1, 1, 16>(p, Mmax, classes, st);
    else if (tiles <= 512) q8_split_launch<1, 2, 8>(p, Mmax, classes, st);
    else q8_split_launch<2, 2, 4>(p, Mmax, classes, st);
  }
  return tde_launch_status();
}

bool q8_rows_ok(int rows, int C, const float* x, int x_cstride, int x_coff, const int8_t* codes, const float* scales) {
  return rows > 0 && rows <= (1 << 30) && C > 0 && C <= Q8_MAXC && x && codes && scales && tde_aligned16(codes) &&
         x_coff >= 0 && (long)x_coff + C <= x_cstride;
}
// 16-byte loads of a channel view (a row's padding up to a multiple of four channels is read)
bool q8_rows_vec(int C, const float* x, int x_cstride, int x_coff) {
  return tde_aligned16(x) && x_cstride % 4 == 0 && x_coff % 4 == 0 && (long)x_coff + (C + 3) / 4 * 4 <= x_cstride;
}
int q8_rows(int rows, int C, const float* x, int x_cstride, int x_coff, int8_t* codes, float* scales, hipStream_t st) {
  const int Cp = q8_row(C), nq = Cp / 4;
  const bool vec = q8_rows_vec(C, x, x_cstride, x_coff);
#define R(LL, QQ, TT)                                                                                                 \
  do {                                                                                                                \
    const long nb = tde_cdiv((long)rows + 1, 256 / LL * TT);                                                          \
    const dim3 grid((unsigned)(nb < (1 << 20) ? nb : 1 << 20));                                                       \
    if (vec)                                                                                                          \
      hipLaunchKernelGGL((q8_rows_kernel<LL, QQ, TT, true>), grid, dim3(256), 0, st, rows, C, Cp, x + x_coff,         \
                         (long)x_cstride, codes, scales);                                                             \
    else                                                                                                              \
      hipLaunchKernelGGL((q8_rows_kernel<LL, QQ, TT, false>), grid, dim3(256), 0, st, rows, C, Cp, x + x_coff,        \
                         (long)x_cstride, codes, scales);                                                             \
  } while (0)
#define W(QQ)                                                                                                          \
  do {                                                                                                                 \
    const long nr = (long)rows + 1;                                                                                    \
    const dim3 grid((unsigned)(nr < 65535 ? nr : 65535), (unsigned)((nr + 65534) / 65535));                            \
    if (vec)                                                                                                           \
      hipLaunchKernelGGL((q8_rows_wide_kernel<QQ, true>), grid, dim3(256), 0, st, (long)rows, C, Cp, x,                \
                         (long)x_cstride, x_coff, codes, scales);                                                      \
    else                                                                                                               \
      hipLaunchKernelGGL((q8_rows_wide_kernel<QQ, false>), grid, dim3(256), 0, st, (long)rows, C, Cp, x,               \
                         (long)x_cstride, x_coff, codes, scales);                                                      \
  } while (0)
  const bool many = rows >= 1 << 15;      // one row per lane group in flight where there are few rows
  if (nq <= 8) { if (many) R(4, 2, 2); else R(4, 2, 1); }
  else if (nq <= 16) { if (many) R(8, 2, 2); else R(16, 1, 1); }
  else if (nq <= 32) { if (many) R(16, 2, 2); else R(32, 1, 1); }
  else if (nq <= 64) { if (many) R(32, 2, 2); else R(64, 1, 1); }
  else if (nq <= 128) R(64, 2, 1);
  else if (nq <= 256) W(1);
  else if (nq <= 512) W(2);
  else W(4);
#undef W
#undef R
  return tde_launch_status();
}

// The small kernel's LDS rows for a geometry, 0: it does not serve.  A block's 16 pixels lie in one image, on at most
// ceil(15 / GW) + 1 rows of its grid, or in several images.
int q8_small_rows(const Q8Conv& p) {
  const int s = p.deconv ? p.os : 1, GH = (p.OH + s - 1) / s, GW = (p.OW + s - 1) / s;
  const long tiles = ((long)tde_cdiv((long)p.N * GH * GW, 16)) * tde_cdiv(p.K, 16) * s * s;
  if (p.Cp % 64 != 0 || p.Cp > 1024 || tiles > 256) return 0;
  const int gh = p.OH / s > 0 ? p.OH / s : 1, gw = p.OW / s > 0 ? p.OW / s : 1;      // the smallest class that has pixels
  const int nty = (p.KH + p.kst - 1) / p.kst, ntx = (p.KW + p.kst - 1) / p.kst;
  const long HW = (long)p.H * p.W;
  long rows;
  if (GH == 1 && gh == 1) rows = (long)(nty < p.H ? nty : p.H) * p.W < (long)(nty - 1) * p.W + 15 * p.is + ntx
                                     ? (long)(nty < p.H ? nty : p.H) * p.W : (long)(nty - 1) * p.W + 15 * p.is + ntx;
  else {
    const long ny = (long)((15 + gw - 1) / gw) * p.is + nty;
    rows = (ny < p.H ? ny : p.H) * p.W;
  }
  if (p.N > 1) {
    const long ni = (15 + gh * gw - 1) / (gh * gw) + 1, all = (ni < p.N ? ni : p.N) * HW;
    if (all > rows) rows = all;
  }
  return rows <= 32 ? (int)rows : 0;
}
int q8_small_launch(const Q8Conv& p, const float* x, long cs, int C, int cap, hipStream_t st) {
  const int s = p.deconv ? p.os : 1, GH = (p.OH + s - 1) / s, GW = (p.OW + s - 1) / s;
  const dim3 grid(tde_cdiv((long)p.N * GH * GW, 16), tde_cdiv(p.K, 16), s * s);
  const Q8Src in{x, cs, C, cap};
  const int lds = (cap + 1) * (p.Cp + 16) + 15 * 1024;
  if (p.Cp <= 256) hipLaunchKernelGGL((q8_small_kernel<1, 4>), grid, dim3(1024), lds, st, p, in);
  else if (p.Cp <= 512) hipLaunchKernelGGL((q8_small_kernel<2, 2>), grid, dim3(1024), lds, st, p, in);
  else hipLaunchKernelGGL((q8_small_kernel<4, 1>), grid, dim3(1024), lds, st, p, in);
  return tde_launch_status();
}

// what the entries check: geometry within int arithmetic, pointers, alignment of codes and scales
bool q8_geometry_ok(const tde_conv_desc_t* d, int cin, int cout) {
  if (d->N <= 0 || d->H <= 0 || d->W <= 0 || d->OH <= 0 || d->OW <= 0 || d->KH <= 0 || d->KW <= 0 || d->stride <= 0 ||
      d->pad_top < 0 || d->pad_left < 0 || d->pad_top >= d->KH || d->pad_left >= d->KW)
    return false;
  if (cin <= 0 || cin > Q8_MAXC || cout <= 0 || cout > 65535 || d->KH > 64 || d->KW > 64 || d->stride > 64) return false;
  const auto fits = [&](int h, int w) { return (long)h * w <= Q8_MAXPIX && (long)d->N * ((long)h * w) <= Q8_MAXPIX; };
  return fits(d->H, d->W) && fits(d->OH, d->OW);      // (the product of three ints may not fit 64 bits)
}
bool q8_args_ok(const tde_conv_desc_t* d, const int8_t* xc, const float* xs, const int8_t* wc, const float* ws, int relu,
                const float* y, int cin, int cout, int ocs, int oco) {
  if (!wc || !ws || !y || !q8_geometry_ok(d, cin, cout)) return false;
  if (ocs <= 0 || oco < 0 || (long)oco + cout > ocs) return false;
  return (relu == 0 || relu == 1) && tde_aligned16(xc) && tde_aligned16(wc) && tde_aligned16(ws) &&
         (reinterpret_cast<uintptr_t>(xs) & 3u) == 0 && (reinterpret_cast<uintptr_t>(y) & 3u) == 0;
}

Q8Conv q8_conv_args(const tde_conv_desc_t* d, const int8_t* x_codes, const float* x_scales, const int8_t* w_codes,
                    const float* w_scales, const float* bias, int relu, float* y) {
  Q8Conv p{};
  p.N = d->N; p.H = d->H; p.W = d->W; p.OH = d->OH; p.OW = d->OW;
  p.Cp = q8_row(d->w_cin); p.K = d->K; p.Kp = q8_cols(d->K);
  p.KH = d->KH; p.KW = d->KW; p.pt = d->pad_top; p.pl = d->pad_left;
  p.is = d->stride; p.os = 1; p.dir = 1; p.kst = 1; p.deconv = 0;
  p.x = x_codes; p.xs = x_scales; p.w = w_codes; p.ws = w_scales; p.bias = bias; p.y = y;
  p.ycs = d->y_cstride; p.yco = d->y_coff; p.relu = relu;
  p.vec = tde_aligned16(y) && p.ycs % 4 == 0 && p.yco % 4 == 0;
  return p;
}
Q8Conv q8_deconv_args(const tde_conv_desc_t* d, const int8_t* x_codes, const float* x_scales, const int8_t* w_codes,
                      const float* w_scales, const float* bias, int relu, float* y_big) {
  Q8Conv p{};
  p.N = d->N; p.H = d->OH; p.W = d->OW; p.OH = d->H; p.OW = d->W;
  p.Cp = q8_row(d->K); p.K = d->C; p.Kp = q8_cols(d->C);
  p.KH = d->KH; p.KW = d->KW; p.pt = d->pad_top; p.pl = d->pad_left;
  p.is = 1; p.os = d->stride; p.dir = -1; p.kst = d->stride; p.deconv = 1;
  p.x = x_codes; p.xs = x_scales; p.w = w_codes; p.ws = w_scales; p.bias = bias; p.y = y_big;
  p.ycs = d->x_cstride; p.yco = d->x_coff; p.relu = relu;
  p.vec = tde_aligned16(y_big) && p.ycs % 4 == 0 && p.yco % 4 == 0;
  return p;
}

// from the fp32 input (its channel view): in one launch, or quantised into codes and scales first (always where the output
// may lie on the input, which a block of one launch could still have to read)
int q8_conv_f32(const Q8Conv& p, const float* x, int C, int cs, int co, int8_t* codes, float* scales, hipStream_t st) {
  TDE_CHECK_ARG(x && co >= 0 && (long)co + C <= cs);
  const int cap = q8_rows_vec(C, x, cs, co) ? q8_small_rows(p) : 0;
  const uintptr_t x0 = reinterpret_cast<uintptr_t>(x), x1 = x0 + (size_t)p.N * p.H * p.W * cs * sizeof(float);
  const uintptr_t y0 = reinterpret_cast<uintptr_t>(p.y), y1 = y0 + (size_t)p.N * p.OH * p.OW * p.ycs * sizeof(float);
  if (cap > 0 && (x1 <= y0 || y1 <= x0)) return q8_small_launch(p, x + co, cs, C, cap, st);
  const int rows = p.N * p.H * p.W;
  TDE_CHECK_ARG(q8_rows_ok(rows, C, x, cs, co, codes, scales));
  const int rc = q8_rows(rows, C, x, cs, co, codes, scales, st);
  return rc != TDE_OK ? rc : q8_conv(p, st);
}

}  // namespace

extern "C" {

int tde_q8_row_bytes(int C) { return C > 0 && C <= Q8_MAXC ? q8_row(C) : 0; }

int tde_q8_rows(int rows, int C, const float* x, int x_cstride, int x_coff, int8_t* codes, float* scales, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(q8_rows_ok(rows, C, x, x_cstride, x_coff, codes, scales));
  return q8_rows(rows, C, x, x_cstride, x_coff, codes, scales, static_cast<hipStream_t>(stream));
}

size_t tde_q8_weights_size(int taps, int cin, int K) {
  if (taps <= 0 || cin <= 0 || cin > Q8_MAXC || K <= 0 || K > 65535) return 0;
  return (size_t)taps * q8_cols(K) * q8_row(cin);
}

int tde_q8_weights(int taps, int cin, int K, int layout, const float* w, int8_t* codes, float* scales, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(tde_q8_weights_size(taps, cin, K) > 0 && taps <= 4096 && (layout == 0 || layout == 1) && w && codes &&
                scales && tde_aligned16(codes));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (layout == 0 && K % 4 == 0 && tde_aligned16(w))
    hipLaunchKernelGGL(q8_weights4_kernel, dim3(q8_cols(K) / 16), dim3(1024), 0, st, taps, cin, K, q8_cols(K), q8_row(cin), w,
                       codes, scales);
  else
    hipLaunchKernelGGL(q8_weights_kernel, dim3(q8_cols(K) / 4), dim3(1024), 0, st, taps, cin, K, q8_cols(K), q8_row(cin),
                       layout, w, codes, scales);
  return tde_launch_status();
}

int tde_q8_conv2d_bias_act(const tde_conv_desc_t* d, const int8_t* x_codes, const float* x_scales,
                           const int8_t* w_codes, const float* w_scales, const float* bias, int relu, float* y,
                           void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(d != nullptr && x_codes && x_scales);
  TDE_CHECK_ARG(q8_args_ok(d, x_codes, x_scales, w_codes, w_scales, relu, y, d->w_cin, d->K, d->y_cstride, d->y_coff));
  return q8_conv(q8_conv_args(d, x_codes, x_scales, w_codes, w_scales, bias, relu, y), static_cast<hipStream_t>(stream));
}

int tde_q8_deconv2d_bias_act(const tde_conv_desc_t* d, const int8_t* x_codes, const float* x_scales,
                             const int8_t* w_codes, const float* w_scales, const float* bias, int relu, float* y_big,
                             void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(d != nullptr && x_codes && x_scales);
  // the virtual conv's x is the output, its y the input
  TDE_CHECK_ARG(q8_args_ok(d, x_codes, x_scales, w_codes, w_scales, relu, y_big, d->K, d->C, d->x_cstride, d->x_coff));
  return q8_conv(q8_deconv_args(d, x_codes, x_scales, w_codes, w_scales, bias, relu, y_big),
                 static_cast<hipStream_t>(stream));
}

int tde_q8_one_launch(const tde_conv_desc_t* d, int deconv) {
  if (!d || !q8_geometry_ok(d, deconv ? d->K : d->w_cin, deconv ? d->C : d->K)) return 0;
  const int cs = deconv ? d->y_cstride : d->x_cstride, co = deconv ? d->y_coff : d->x_coff;
  if (!q8_rows_vec(deconv ? d->K : d->w_cin, nullptr, cs, co)) return 0;
  const Q8Conv p = deconv ? q8_deconv_args(d, nullptr, nullptr, nullptr, nullptr, nullptr, 0, nullptr)
                          : q8_conv_args(d, nullptr, nullptr, nullptr, nullptr, nullptr, 0, nullptr);
  return q8_small_rows(p) > 0;
}

int tde_q8_conv2d_f32_bias_act(const tde_conv_desc_t* d, const float* x, int8_t* x_codes, float* x_scales,
                               const int8_t* w_codes, const float* w_scales, const float* bias, int relu, float* y,
                               void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(d != nullptr);
  TDE_CHECK_ARG(q8_args_ok(d, x_codes, x_scales, w_codes, w_scales, relu, y, d->w_cin, d->K, d->y_cstride, d->y_coff));
  return q8_conv_f32(q8_conv_args(d, x_codes, x_scales, w_codes, w_scales, bias, relu, y), x, d->w_cin, d->x_cstride,
                     d->x_coff, x_codes, x_scales, static_cast<hipStream_t>(stream));
}

int tde_q8_deconv2d_f32_bias_act(const tde_conv_desc_t* d, const float* x_small, int8_t* x_codes, float* x_scales,
                                 const int8_t* w_codes, const float* w_scales, const float* bias, int relu, float* y_big,
                                 void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(d != nullptr);
  TDE_CHECK_ARG(q8_args_ok(d, x_codes, x_scales, w_codes, w_scales, relu, y_big, d->K, d->C, d->x_cstride, d->x_coff));
  return q8_conv_f32(q8_deconv_args(d, x_codes, x_scales, w_codes, w_scales, bias, relu, y_big), x_small, d->K,
                     d->y_cstride, d->y_coff, x_codes, x_scales, static_cast<hipStream_t>(stream));
}

}  // extern "C"
