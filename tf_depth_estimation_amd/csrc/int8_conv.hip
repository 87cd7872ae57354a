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
#include "tde_common.h"

#include <type_traits>

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));

// code bytes of a row of C channels: the reduction depth of one matrix instruction (32 or 64)
inline int q8_row(int C) { return C <= 32 ? 32 : (C + 63) / 64 * 64; }
inline int q8_cols(int K) { return (K + 15) / 16 * 16; }
constexpr int Q8_MAXC = 4096;

__device__ __forceinline__ float q8_scale(unsigned amax_bits) {
  return amax_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(amax_bits) / 127.f;
}

// rne(127 x / a), exact.  The fp32 estimate t = x * (127 / a) is off by less than 4e-5 (three roundings of at most 127),
// so unless t lies that close to a half-integer its rounding is the quotient's.  Near one (1 element in 10^4) the fp64
// remainder 254 x - 2 q a (exact: 24-bit factors) decides, and breaks a tie to even.  a: finite maximum, |x| <= a.
struct Q8Div {
  double a;
  float inv;
  int mode;          // 0: the row is zero or not finite, 1: fp32 estimate, 2: fp64 division (1 / a may be no normal number)
};
__device__ __forceinline__ Q8Div q8_div(unsigned amax_bits) {
  Q8Div d;
  const float a = __uint_as_float(amax_bits);
  d.a = (double)a;
  d.inv = 0.f;
  d.mode = amax_bits == 0 || amax_bits >= 0x7f800000u ? 0 : (a >= 0x1p-100f && a <= 0x1p100f ? 1 : 2);
  if (d.mode == 1) d.inv = 127.f * __builtin_amdgcn_rcpf(a);
  return d;
}
__device__ __noinline__ int q8_code_exact(float x, double a) {
  const double xd = 127.0 * (double)x;
  int q = (int)rint(xd / a);
  const double r = 2.0 * fma(-(double)q, a, xd);
  if (r > a || (r == a && (q & 1))) ++q;
  if (r < -a || (r == -a && (q & 1))) --q;
  return q;
}
// codes of four channels, packed
__device__ __forceinline__ int q8_code4(const f4& x, const Q8Div& d) {
  f4 q;
  bool near = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float t = x[j] * d.inv;
    q[j] = rintf(t);
    near |= fabsf(fabsf(t - q[j]) - 0.5f) < 5e-5f;
  }
  int p = 0;
  if (d.mode == 2 || (near && d.mode == 1)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p |= (q8_code_exact(x[j], d.a) & 0xff) << (8 * j);
    return p;
  }
  if (d.mode == 0) return 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) p |= ((int)q[j] & 0xff) << (8 * j);
  return p;
}

// ---- rows: L lanes per row (a power of two <= 64), QPL quads of channels per lane held in registers; VEC: 16-byte loads
template <int L, int QPL, bool VEC>
__global__ void __launch_bounds__(256) q8_rows_kernel(long rows, int C, int Cp, const float* x, long cs, int co,
                                                      int8_t* codes, float* scales) {
  const int l = threadIdx.x % L;
  const long row = (long)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row > rows) return;
  const float* px = x + row * cs + co;
  f4 v[QPL];
  unsigned am = 0;
#pragma unroll
  for (int i = 0; i < QPL; ++i) {
    const int c = 4 * (l + i * L);
    v[i] = f4{0.f, 0.f, 0.f, 0.f};
    if (row < rows && c < C) {
      if (VEC) {
        v[i] = *reinterpret_cast<const f4*>(px + c);
#pragma unroll
        for (int j = 1; j < 4; ++j)
          if (c + j >= C) v[i][j] = 0.f;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < C) v[i][j] = px[c + j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) am = max(am, __float_as_uint(v[i][j]) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) am = max(am, (unsigned)__shfl_xor((int)am, o, 64));
  const Q8Div d = q8_div(am);
#pragma unroll
  for (int i = 0; i < QPL; ++i) {
    const int c = 4 * (l + i * L);
    if (c < Cp) *reinterpret_cast<int*>(codes + row * Cp + c) = q8_code4(v[i], d);
  }
  if (l == 0) scales[row] = q8_scale(am);      // (row `rows`: no channel was read, scale 0)
}

// ---- weights: one block per output channel (padding channels write zeros)
__global__ void __launch_bounds__(256) q8_weights_kernel(int taps, int cin, int K, int Kp, int Cp, int layout,
                                                         const float* w, int8_t* codes, float* scales) {
  __shared__ unsigned sh[4];
  const int k = blockIdx.x;
  unsigned am = 0;
  if (k < K)
    for (int i = threadIdx.x; i < taps * cin; i += 256) {
      const int t = i / cin, c = i - t * cin;
      const float v = layout == 0 ? w[((long)t * cin + c) * K + k] : w[((long)t * K + k) * cin + c];
      am = max(am, __float_as_uint(v) & 0x7fffffffu);
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) am = max(am, (unsigned)__shfl_xor((int)am, o, 64));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = am;
  __syncthreads();
  am = max(max(sh[0], sh[1]), max(sh[2], sh[3]));
  const Q8Div d = q8_div(am);
  for (int i = threadIdx.x; i < taps * Cp / 4; i += 256) {
    const int t = 4 * i / Cp, c = 4 * i - t * Cp;
    f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k < K && c + j < cin)
        v[j] = layout == 0 ? w[((long)t * cin + c + j) * K + k] : w[((long)t * K + k) * cin + c + j];
    *reinterpret_cast<int*>(codes + ((long)t * Kp + k) * Cp + c) = q8_code4(v, d);
  }
  if (threadIdx.x == 0) scales[k] = q8_scale(am);
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

// WK waves split the (tap, channel chunk) steps of a tile of 16 TM channels x 16 TN pixels and add their fp32 sums through
// LDS in wave order; WP groups of WK waves take neighbouring pixel tiles.  Fragments come straight from the caches:
// a lane's 16 (8) bytes are its row's k-quarter, so a fragment is 16 segments of 64 (32) contiguous bytes.
template <int TM, int TN, int KC, int WK, int WP>
__global__ void __launch_bounds__(64 * WK * WP) q8_conv_kernel(const Q8Conv p) {
  using F = typename Q8Frag<KC>::T;
  __shared__ f4 red[WK > 1 ? WP * (WK - 1) * TM * TN * 64 : 1];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, wk = wv % WK, wp = wv / WK;
  const int r16 = lane & 15, kq = lane >> 4;
  const Q8Class cl = q8_class(p, blockIdx.z);
  const int m0 = (blockIdx.x * WP + wp) * 16 * TN, n0 = blockIdx.y * 16 * TM;
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
  int s = (int)((long)steps * wk / WK);
  const int s1 = (int)((long)steps * (wk + 1) / WK);
  while (s < s1) {
    const int t = s / nch, ch0 = s - t * nch, ch1 = min(nch, ch0 + s1 - s);
    const int ty = t / cl.ntx, tx = t - ty * cl.ntx;
    const long wtap = ((long)(cl.ky0 + p.kst * ty) * p.KW + cl.kx0 + p.kst * tx) * p.Kp * p.Cp;
    const int8_t* xr[TN];
    float xs[TN];
#pragma unroll
    for (int b = 0; b < TN; ++b) {
      const int yy = iy[b] + p.dir * ty, xx = ix[b] + p.dir * tx;
      const bool in = (unsigned)yy < (unsigned)p.H && (unsigned)xx < (unsigned)p.W;
      const long pix = in ? pb[b] + (long)yy * p.W + xx : zero_row;
      xr[b] = p.x + pix * p.Cp + kq * (KC / 4);
      xs[b] = p.xs[pix];
    }
    i4 ia[TM][TN];
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b) ia[a][b] = i4{0, 0, 0, 0};
    for (int ch = ch0; ch < ch1; ++ch) {
      F fa[TM], fb[TN];
#pragma unroll
      for (int a = 0; a < TM; ++a) fa[a] = *reinterpret_cast<const F*>(wrow[a] + wtap + ch * KC);
#pragma unroll
      for (int b = 0; b < TN; ++b) fb[b] = *reinterpret_cast<const F*>(xr[b] + ch * KC);
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) ia[a][b] = Q8Frag<KC>::mfma(fa[a], fb[b], ia[a][b]);
    }
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
      for (int b = 0; b < TN; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[a][b][j] = fmaf((float)ia[a][b][j], xs[b], acc[a][b][j]);
    s += ch1 - ch0;
  }

  if (WK > 1) {
    f4* mine = red + wp * (WK - 1) * TM * TN * 64;
    if (wk > 0)
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) mine[((wk - 1) * TM * TN + a * TN + b) * 64 + lane] = acc[a][b];
    __syncthreads();
    if (wk > 0) return;
    for (int w = 0; w < WK - 1; ++w)
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) acc[a][b] += mine[(w * TM * TN + a * TN + b) * 64 + lane];
  }

#pragma unroll
  for (int b = 0; b < TN; ++b) {
    const int m = m0 + 16 * b + r16;
    if (m >= cl.M) continue;
    const int hw = cl.GH * cl.GW, n = m / hw, r = m - n * hw, i = r / cl.GW, j = r - i * cl.GW;
    float* py = p.y + (((long)n * p.OH + i * p.os + cl.py) * p.OW + j * p.os + cl.px) * p.ycs + p.yco;
#pragma unroll
    for (int a = 0; a < TM; ++a) {
      const int k = n0 + 16 * a + 4 * kq;
      if (k >= p.K) continue;
      const f4 ws = *reinterpret_cast<const f4*>(p.ws + k);       // (scales are padded to Kp)
      f4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = fmaf(acc[a][b][e], ws[e], p.bias && k + e < p.K ? p.bias[k + e] : 0.f);
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
  }
}

template <int TM, int TN, int WK, int WP>
void q8_launch(const Q8Conv& p, long Mmax, int classes, hipStream_t st) {
  const dim3 grid(tde_cdiv(Mmax, 16 * TN * WP), tde_cdiv(p.K, 16 * TM), classes);
  if (p.Cp % 64 == 0)
    hipLaunchKernelGGL((q8_conv_kernel<TM, TN, 64, WK, WP>), grid, dim3(64 * WK * WP), 0, st, p);
  else
    hipLaunchKernelGGL((q8_conv_kernel<TM, TN, 32, WK, WP>), grid, dim3(64 * WK * WP), 0, st, p);
}

int q8_conv(Q8Conv p, hipStream_t st) {
  const int s = p.deconv ? p.os : 1;
  const long Mmax = (long)p.N * ((p.OH + s - 1) / s) * ((p.OW + s - 1) / s);
  if (Mmax > (1 << 30)) return TDE_ERR_UNSUPPORTED;
  const int classes = s * s;
  const long tiles = ((Mmax + 15) / 16) * ((p.K + 15) / 16) * classes;      // 16 x 16 tiles
  if (tiles <= 2048) q8_launch<1, 1, 16, 1>(p, Mmax, classes, st);
  else if (tiles <= 16384) q8_launch<2, 2, 4, 1>(p, Mmax, classes, st);
  else if (p.K <= 16) q8_launch<1, 4, 1, 4>(p, Mmax, classes, st);
  else if (p.K <= 32) q8_launch<2, 4, 1, 4>(p, Mmax, classes, st);
  else q8_launch<4, 4, 1, 4>(p, Mmax, classes, st);
  return tde_launch_status();
}

// what both entries check: geometry within int arithmetic, pointers, alignment of codes and scales
bool q8_args_ok(const tde_conv_desc_t* d, const int8_t* xc, const float* xs, const int8_t* wc, const float* ws, int relu,
                const float* y, int cin, int cout, int ocs, int oco) {
  if (!d || !xc || !xs || !wc || !ws || !y) return false;
  if (d->N <= 0 || d->H <= 0 || d->W <= 0 || d->OH <= 0 || d->OW <= 0 || d->KH <= 0 || d->KW <= 0 || d->stride <= 0 ||
      d->pad_top < 0 || d->pad_left < 0 || d->pad_top >= d->KH || d->pad_left >= d->KW)
    return false;
  if (cin <= 0 || cin > Q8_MAXC || cout <= 0 || cout > 65535 || d->KH > 64 || d->KW > 64 || d->stride > 64) return false;
  if ((long)d->N * d->H * d->W > (1 << 30) || (long)d->N * d->OH * d->OW > (1 << 30)) return false;
  if (ocs <= 0 || oco < 0 || oco + cout > ocs) return false;
  return (relu == 0 || relu == 1) && tde_aligned16(xc) && tde_aligned16(wc) && tde_aligned16(ws) &&
         (reinterpret_cast<uintptr_t>(xs) & 3u) == 0 && (reinterpret_cast<uintptr_t>(y) & 3u) == 0;
}

}  // namespace

extern "C" {

int tde_q8_row_bytes(int C) { return C > 0 && C <= Q8_MAXC ? q8_row(C) : 0; }

int tde_q8_rows(int rows, int C, const float* x, int x_cstride, int x_coff, int8_t* codes, float* scales, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(rows > 0 && rows <= (1 << 30) && C > 0 && C <= Q8_MAXC && x && codes && scales && tde_aligned16(codes) &&
                x_coff >= 0 && x_coff + C <= x_cstride);
  const int Cp = q8_row(C), nq = Cp / 4;
  const bool vec = tde_aligned16(x) && x_cstride % 4 == 0 && x_coff % 4 == 0 && x_coff + (C + 3) / 4 * 4 <= x_cstride;
  hipStream_t st = static_cast<hipStream_t>(stream);
#define R(LL, QQ)                                                                                                     \
  do {                                                                                                                \
    const dim3 grid(tde_cdiv((long)rows + 1, 256 / LL));                                                              \
    if (vec)                                                                                                          \
      hipLaunchKernelGGL((q8_rows_kernel<LL, QQ, true>), grid, dim3(256), 0, st, (long)rows, C, Cp, x, (long)x_cstride, \
                         x_coff, codes, scales);                                                                      \
    else                                                                                                              \
      hipLaunchKernelGGL((q8_rows_kernel<LL, QQ, false>), grid, dim3(256), 0, st, (long)rows, C, Cp, x,               \
                         (long)x_cstride, x_coff, codes, scales);                                                     \
  } while (0)
  if (nq <= 8) R(8, 1);
  else if (nq <= 16) R(16, 1);
  else if (nq <= 32) R(32, 1);
  else if (nq <= 64) R(64, 1);
  else if (nq <= 128) R(64, 2);
  else if (nq <= 256) R(64, 4);
  else if (nq <= 512) R(64, 8);
  else R(64, 16);
#undef R
  return tde_launch_status();
}

size_t tde_q8_weights_size(int taps, int cin, int K) {
  if (taps <= 0 || cin <= 0 || cin > Q8_MAXC || K <= 0 || K > 65535) return 0;
  return (size_t)taps * q8_cols(K) * q8_row(cin);
}

int tde_q8_weights(int taps, int cin, int K, int layout, const float* w, int8_t* codes, float* scales, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(tde_q8_weights_size(taps, cin, K) > 0 && taps <= 4096 && (layout == 0 || layout == 1) && w && codes &&
                scales && tde_aligned16(codes));
  hipLaunchKernelGGL(q8_weights_kernel, dim3(q8_cols(K)), dim3(256), 0, static_cast<hipStream_t>(stream), taps, cin, K,
                     q8_cols(K), q8_row(cin), layout, w, codes, scales);
  return tde_launch_status();
}

int tde_q8_conv2d_bias_act(const tde_conv_desc_t* d, const int8_t* x_codes, const float* x_scales,
                           const int8_t* w_codes, const float* w_scales, const float* bias, int relu, float* y,
                           void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(d != nullptr);
  TDE_CHECK_ARG(q8_args_ok(d, x_codes, x_scales, w_codes, w_scales, relu, y, d->w_cin, d->K, d->y_cstride, d->y_coff));
  Q8Conv p{};
  p.N = d->N; p.H = d->H; p.W = d->W; p.OH = d->OH; p.OW = d->OW;
  p.Cp = q8_row(d->w_cin); p.K = d->K; p.Kp = q8_cols(d->K);
  p.KH = d->KH; p.KW = d->KW; p.pt = d->pad_top; p.pl = d->pad_left;
  p.is = d->stride; p.os = 1; p.dir = 1; p.kst = 1; p.deconv = 0;
  p.x = x_codes; p.xs = x_scales; p.w = w_codes; p.ws = w_scales; p.bias = bias; p.y = y;
  p.ycs = d->y_cstride; p.yco = d->y_coff; p.relu = relu;
  p.vec = tde_aligned16(y) && p.ycs % 4 == 0 && p.yco % 4 == 0;
  return q8_conv(p, static_cast<hipStream_t>(stream));
}

int tde_q8_deconv2d_bias_act(const tde_conv_desc_t* d, const int8_t* x_codes, const float* x_scales,
                             const int8_t* w_codes, const float* w_scales, const float* bias, int relu, float* y_big,
                             void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(d != nullptr);
  // the virtual conv's x is the output, its y the input
  TDE_CHECK_ARG(q8_args_ok(d, x_codes, x_scales, w_codes, w_scales, relu, y_big, d->K, d->C, d->x_cstride, d->x_coff));
  Q8Conv p{};
  p.N = d->N; p.H = d->OH; p.W = d->OW; p.OH = d->H; p.OW = d->W;
  p.Cp = q8_row(d->K); p.K = d->C; p.Kp = q8_cols(d->C);
  p.KH = d->KH; p.KW = d->KW; p.pt = d->pad_top; p.pl = d->pad_left;
  p.is = 1; p.os = d->stride; p.dir = -1; p.kst = d->stride; p.deconv = 1;
  p.x = x_codes; p.xs = x_scales; p.w = w_codes; p.ws = w_scales; p.bias = bias; p.y = y_big;
  p.ycs = d->x_cstride; p.yco = d->x_coff; p.relu = relu;
  p.vec = tde_aligned16(y_big) && p.ycs % 4 == 0 && p.yco % 4 == 0;
  return q8_conv(p, static_cast<hipStream_t>(stream));
}

}  // extern "C"
