// The 8-bit tape of training BatchNorm + ReLU (include/tde.h, "8-bit activations" (2)).
//
// Forward: per channel and row group mean / variance of z (fp64), u = (z - mean) * invstd + beta (fp64),
// y = relu(u), and u kept as one byte per element: blocks of 64 channels of a row share a = max|u| (fp64), s = (float)a / 128
// and the mid-rise code floor(128 |u| / a) with u's sign folded in (q >= 0 iff u > 0; value (q + 1/2) s).
// Backward: g = dy [q >= 0], xhat = (q + 1/2) s - beta, dz = invstd (g - mean g - xhat mean(g xhat)).
//
// u is evaluated in fp64 because a code next to a step's border flips with the last bits of u: with fp64 the codes are
// those of the definition (tape_code4).  fp64 FMAs run at the fp32 rate here, so the passes stay bound by memory.
//
// Lanes: a row's block of 64 channels is one 16-lane DPP row, four channels per lane (narrower layers use 1-8 lanes per
// row), so max|u| is four DPP moves, a row's z / dy is one 16-byte and its codes one 4-byte access per lane.
#include "int8_common.h"

#include "bn_internal.h"

namespace {

typedef double d4 __attribute__((ext_vector_type(4)));

// lanes that hold one row's channel block: a power of two >= min(C, 64) / 4
int tape_lanes(int C) {
  int l = 1;
  while (l < 16 && 4 * l < C) l *= 2;
  return l;
}

// codes of four u of a block with maximum a = max|u| and scale s = (float)a / 128, packed: the exact floor(128 |u| / a) clamped
// to 127, sign folded in (~q for u <= 0).  The fp32 estimate t = |u| / s is off by less than 4e-5 (|u|, a and the product are
// rounded by half a step each, the reciprocal is off by up to one: 5 * 2^-24 of at most 128), so unless t lies that close to
// an integer its floor is the quotient's; near one (1 element in 10^4) the fp64 remainder against the unrounded a decides,
// which the lanes of a row exchange only then.  (Against the rounded s one code in 10^6 is off by one.)  Estimates past 127.25
// are set there: they are clamped to 127 anyway, and every block's maximum, at 128, would take the exact path.
__device__ __noinline__ int tape_code_exact(double u, double a, float s) {
  int q = 0;
  if (a > 0.0 && s == s) {             // (a block of zeros, or one that is not finite: 0 / -1)
    const double au = 128.0 * fabs(u);
    q = (int)fmin(floor(au / a), 127.0);
    const double r = fma(-(double)q, a, au);
    if (r < 0.0) --q;
    if (r >= a && q < 127) ++q;
  }
  return u > 0.0 ? q : -1 - q;
}
// maximum over the aligned group of L lanes, in every lane; all L lanes must be active
template <int L>
__device__ __forceinline__ double group_dmax(double v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v = fmax(v, __shfl_xor(v, o, 64));
  return v;
}
template <int L>
__device__ __forceinline__ int tape_code4(const d4& u, const f4& uf, float s) {
  bool near = !(s >= 0x1p-100f);       // (1 / s may be no normal number)
  const float inv = __builtin_amdgcn_rcpf(s);
  f4 q;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float t = fminf(fabsf(uf[j]) * inv, 127.25f);
    q[j] = floorf(t);
    near |= fabsf((t - q[j]) - 0.5f) > 0.49995f && t > 0.5f;
  }
  unsigned p = put_byte<0>(q[0], 0);
  p = put_byte<1>(q[1], p);
  p = put_byte<2>(q[2], p);
  p = put_byte<3>(q[3], p);
#pragma unroll
  for (int j = 0; j < 4; ++j) p ^= u[j] > 0.0 ? 0u : 0xffu << (8 * j);
  if (__any(near)) {                   // (uniform over the wave: every lane of a row's group takes part in the exchange)
    const double a = group_dmax<L>(fmax(fmax(fabs(u[0]), fabs(u[1])), fmax(fabs(u[2]), fabs(u[3]))));
    if (near) {
      p = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) p |= (unsigned)(tape_code_exact(u[j], a, s) & 0xff) << (8 * j);
    }
  }
  return (int)p;
}

// scale of a block from the bits of max|u| (NaN and infinity order above every finite value)
__device__ __forceinline__ float tape_scale(unsigned amax_bits) {
  return amax_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(amax_bits) * 0.0078125f;
}

__device__ __forceinline__ float tape_value(int packed, int j, float s) {
  return ((float)(int8_t)(packed >> (8 * j)) + 0.5f) * s;
}

// y (4 channels), packed codes and the block scale of one row; every lane of the row's group calls it (lanes past C
// with u = 0)
template <int L>
__device__ __forceinline__ void tape_row(const d4& u, f4& y, int& packed, float& s) {
  unsigned am = 0;
  f4 uf;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uf[j] = (float)u[j];
    y[j] = uf[j] < 0.f ? 0.f : uf[j];
    am = max(am, abs_bits(uf[j]));
  }
  s = tape_scale(group_umax<L>(am));
  packed = tape_code4<L>(u, uf, s);
}

struct TapeFwd {
  int Mg, C, NB, G;          // rows per group, channels, 64-channel blocks, groups
  const float *z, *beta;
  double Mt, invM;           // rows per group over all replicas
  float eps, decay;
  int bessel;
  float *mm, *mv, *save_mean, *save_invstd;
  float* y;
  int ycs, yco;
  int8_t* codes;
  float* scales;
};

// mean (a true quotient: a constant channel's mean is its value, so u = beta there), variance, 1 / sqrt(var + eps): the
// estimate of v_rsq_f64 and two Newton steps, off by a last bit or two, for a quarter of the instructions of sqrt and divide
__device__ __forceinline__ void tape_stats(double s0, double s1, double Mt, double invM, float eps, double& mean,
                                           double& var, double& is) {
  mean = s0 / Mt;
  var = s1 * invM - mean * mean;
  if (var < 0) var = 0;
  const double x = var + (double)eps;
  double y = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(0.5 * y, fma(-x * y, y, 1.0), y);
  is = x > 0.0 && x < 1e300 ? y : 1.0 / sqrt(x);          // (zero, infinity and NaN: as the formula)
}

// statistics and moving averages of channel c of every group, groups in order
__device__ __forceinline__ void tape_publish(const TapeFwd& p, const double* sums, int c) {
  float m0 = p.mm ? p.mm[c] : 0.f, v0 = p.mm ? p.mv[c] : 0.f;
  for (int g = 0; g < p.G; ++g) {
    double mean, var, is;
    tape_stats(sums[(long)g * 2 * p.C + c], sums[(long)g * 2 * p.C + p.C + c], p.Mt, p.invM, p.eps, mean, var, is);
    p.save_mean[(long)g * p.C + c] = (float)mean;
    p.save_invstd[(long)g * p.C + c] = (float)is;
    const double vu = (p.bessel && p.Mt > 1) ? var * p.Mt / (p.Mt - 1) : var;
    m0 -= (m0 - (float)mean) * (1.f - p.decay);
    v0 -= (v0 - (float)vu) * (1.f - p.decay);
  }
  if (p.mm) { p.mm[c] = m0; p.mv[c] = v0; }
}

// ---- sums of a row chunk: part[chunk][2][C].  MODE 0: z, z^2; MODE 1: g, g xhat.  Grid (chunk, 64-channel block);
// rowlane order and the tree below are fixed, so the sums are too.  Bound by memory where there are many rows: MODE 0
// 1572864 x 16 17.5 us (5.7 TB/s), MODE 1 393216 x 32 of a 68-channel dy 18.5 us (its 128-byte pieces lie over two lines).
struct TapeSums {
  int C, NB, per_g, rpc, Mg;       // chunks per group, rows per chunk, rows per group
  const float* z;
  const int8_t* codes;
  const float *scales, *beta, *dy;
  int dycs, dyco;
  double* part;
};

constexpr int SUM_RB = 4;          // rows in flight per lane

template <int L, int MODE>
__global__ void __launch_bounds__(256) tape_sums_kernel(const TapeSums p) {
  constexpr int R = 256 / L;
  __shared__ double sh[4][L][8];
  const int tid = threadIdx.x, l = tid % L, rl = tid / L, b = blockIdx.y;
  const int c = 64 * b + 4 * l;
  const bool on = c < p.C;
  const int g = blockIdx.x / p.per_g, k = blockIdx.x - g * p.per_g;
  const long base = (long)g * p.Mg;
  const int r0 = k * p.rpc, r1 = min(p.Mg, r0 + p.rpc);
  d4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
  if (on) {
    f4 bt = {0, 0, 0, 0};
    if (MODE == 1) bt = *reinterpret_cast<const f4*>(p.beta + c);
    for (int rb = r0 + rl; rb < r1; rb += SUM_RB * R) {
      f4 v[SUM_RB];
      int q[SUM_RB];
      float s[SUM_RB];
#pragma unroll
      for (int i = 0; i < SUM_RB; ++i) {
        const int r = rb + i * R;
        const long row = base + r;
        const bool ok = r < r1;
        if (MODE == 0) {
          v[i] = ok ? *reinterpret_cast<const f4*>(p.z + row * p.C + c) : f4{0.f, 0.f, 0.f, 0.f};
        } else {
          v[i] = ok ? *reinterpret_cast<const f4*>(p.dy + row * p.dycs + p.dyco + c) : f4{0.f, 0.f, 0.f, 0.f};
          q[i] = ok ? *reinterpret_cast<const int*>(p.codes + row * p.C + c) : -1;
          s[i] = ok ? p.scales[row * p.NB + b] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < SUM_RB; ++i) {
        if (MODE == 1 && rb + i * R >= r1) break;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (MODE == 0) {
            const double zd = (double)v[i][j];
            s0[j] += zd;
            s1[j] = fma(zd, zd, s1[j]);
          } else {
            const double xh = (double)(tape_value(q[i], j, s[i]) - bt[j]);
            const double gd = (int8_t)(q[i] >> (8 * j)) >= 0 ? (double)v[i][j] : 0.0;
            s0[j] += gd;
            s1[j] = fma(gd, xh, s1[j]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = L; o < 64; o <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s0[j] += __shfl_xor(s0[j], o, 64);
      s1[j] += __shfl_xor(s1[j], o, 64);
    }
  const int lane = tid & 63, wv = tid >> 6;
  if (lane < L)
#pragma unroll
    for (int j = 0; j < 4; ++j) { sh[wv][l][j] = s0[j]; sh[wv][l][4 + j] = s1[j]; }
  __syncthreads();
  if (tid < 8 * L) {
    const int ll = tid >> 3, j = tid & 7, cc = 64 * b + 4 * ll + (j & 3);
    if (cc < p.C)
      p.part[(long)blockIdx.x * 2 * p.C + (j >> 2) * p.C + cc] =
          (sh[0][ll][j] + sh[1][ll][j]) + (sh[2][ll][j] + sh[3][ll][j]);
  }
}

// part [G * per_g][2C] -> sums [G][2C] (and a copy): block = 8 columns x 128 stripes, up to 8 chunks per lane in flight;
// grid (columns, group).  Latency: 3.2 us for 416 chunks, 4.6 for 1024.
__global__ void __launch_bounds__(1024) tape_finalize_kernel(int C2, int per_g, const double* part, double* sums,
                                                             double* copy) {
  __shared__ double sh[128][8];
  const int col = threadIdx.x & 7, st = threadIdx.x >> 3, cc = blockIdx.x * 8 + col;
  const double* pp = part + (long)blockIdx.y * per_g * C2;
  double a = 0;
  if (cc < C2)
    for (int k0 = st; k0 < per_g; k0 += 1024) {
      double v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = k0 + 128 * u < per_g ? pp[(long)(k0 + 128 * u) * C2 + cc] : 0.0;
      a += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
  sh[st][col] = a;
  __syncthreads();
  if (threadIdx.x < 64) {          // one wave: 8 columns x 8 lanes of 16 stripes
    const int part8 = threadIdx.x >> 3;
    double s = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += sh[part8 * 16 + k][col];
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
    if (threadIdx.x < 8 && cc < C2) {
      sums[(long)blockIdx.y * C2 + cc] = s;
      if (copy) copy[(long)blockIdx.y * C2 + cc] = s;
    }
  }
}

constexpr int APPLY_RB = 4;        // rows in flight per lane

// Row lanes of the apply passes: a row is NB * L lanes (NB 64-channel blocks), 256 / (NB * L) rows per step, the next step's
// loads in flight under this one's arithmetic.  1572864 x 16 38 us (6.1 TB/s of reads and writes; the VALU is busy 64 %).
template <int L>
__global__ void __launch_bounds__(256) tape_fwd_apply_kernel(const TapeFwd p, const double* sums, int rpb) {
  const int nl = p.NB * L, R = 256 / nl;
  const int rl = threadIdx.x / nl, q = threadIdx.x - rl * nl;
  if (rl >= R) return;
  const int b = q / L, c = 4 * q, g = blockIdx.y;
  const bool on = c < p.C;
  const long base = (long)g * p.Mg;
  const int r0 = blockIdx.x * rpb, r1 = min(p.Mg, r0 + rpb);
  // row of step i: uniform row rb + i R (addresses in scalar registers) + this lane's rl (32-bit offsets, but in y, whose
  // pixel stride may be any int)
  const unsigned zo = rl * p.C + c, so = rl * p.NB + b;
  const long yo = (long)rl * p.ycs + c;
  f4 v[APPLY_RB];
  auto load = [&](int rb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < APPLY_RB; ++i) {
      v[i] = f4{0.f, 0.f, 0.f, 0.f};
      if (on && rb + i * R + rl < r1) v[i] = *reinterpret_cast<const f4*>(p.z + (base + rb + i * R) * p.C + zo);
    }
  };
  load(r0);                            // in flight while the statistics are evaluated
  d4 mu = {0, 0, 0, 0}, is = {0, 0, 0, 0}, bt = {0, 0, 0, 0};
  if (on) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      double m, var, i;
      tape_stats(sums[(long)g * 2 * p.C + c + j], sums[(long)g * 2 * p.C + p.C + c + j], p.Mt, p.invM, p.eps, m, var, i);
      mu[j] = m; is[j] = i; bt[j] = (double)p.beta[c + j];
      if (blockIdx.x == 0 && g == 0 && rl == 0) tape_publish(p, sums, c + j);
    }
  }
  for (int rb = r0; rb < r1; rb += APPLY_RB * R) {
    f4 w[APPLY_RB];
#pragma unroll
    for (int i = 0; i < APPLY_RB; ++i) w[i] = v[i];
    if (rb + APPLY_RB * R < r1) load(rb + APPLY_RB * R);
#pragma unroll
    for (int i = 0; i < APPLY_RB; ++i) {
      if (rb + i * R + rl >= r1) break;
      const long row = base + rb + i * R;
      d4 u;
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = fma((double)w[i][j] - mu[j], is[j], bt[j]);
      f4 y;
      int packed;
      float s;
      tape_row<L>(u, y, packed, s);
      if (on) {
        tde_st(reinterpret_cast<f4*>(p.y + row * p.ycs + p.yco + yo), y);
        *reinterpret_cast<int*>(p.codes + row * p.C + zo) = packed;
        if (q % L == 0) p.scales[row * p.NB + so] = s;
      }
    }
  }
}

constexpr int SMALL_NT = 512;      // threads of the one-launch kernels (1024 with 8 rows a lane spill: 18 us against 6.5)
constexpr int SMALL_RB = 8;        // most rows a lane of theirs holds

// Few rows (Mg <= SMALL_RB * SMALL_NT / L): one block per 64-channel block keeps its columns of z in registers, so statistics,
// y and the tape are one launch and z is read once.  96 x 512: 6.5 us, the latency of one load, two barriers and the fp64 steps.
template <int L, int RB>
__global__ void __launch_bounds__(SMALL_NT) tape_fwd_small_kernel(const TapeFwd p) {
  constexpr int R = SMALL_NT / L, NW = SMALL_NT / 64;
  __shared__ double sh[NW][L][8];
  __shared__ double tot[L][8];
  const int tid = threadIdx.x, l = tid % L, rl = tid / L, b = blockIdx.x, lane = tid & 63, wv = tid >> 6;
  const int c = 64 * b + 4 * l;
  const bool on = c < p.C;
  d4 bt = {0, 0, 0, 0};
  float m0[4] = {0, 0, 0, 0}, v0[4] = {0, 0, 0, 0};
  if (on)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bt[j] = (double)p.beta[c + j];
      if (p.mm && rl == 0) { m0[j] = p.mm[c + j]; v0[j] = p.mv[c + j]; }
    }
  for (int g = 0; g < p.G; ++g) {
    const long base = (long)g * p.Mg;
    f4 v[RB];
    d4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int r = rl + i * R;
      v[i] = on && r < p.Mg ? *reinterpret_cast<const f4*>(p.z + (base + r) * p.C + c) : f4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double zd = (double)v[i][j];
        s0[j] += zd;
        s1[j] = fma(zd, zd, s1[j]);
      }
#pragma unroll
    for (int o = L; o < 64; o <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s0[j] += __shfl_xor(s0[j], o, 64);
        s1[j] += __shfl_xor(s1[j], o, 64);
      }
    if (lane < L)
#pragma unroll
      for (int j = 0; j < 4; ++j) { sh[wv][l][j] = s0[j]; sh[wv][l][4 + j] = s1[j]; }
    __syncthreads();
    if (tid < 8 * L) {
      double s = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) s += sh[w][tid >> 3][tid & 7];
      tot[tid >> 3][tid & 7] = s;
    }
    __syncthreads();
    d4 mu = {0, 0, 0, 0}, is = {0, 0, 0, 0};
    if (on)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        double m, var, i;
        tape_stats(tot[l][j], tot[l][4 + j], p.Mt, p.invM, p.eps, m, var, i);
        mu[j] = m; is[j] = i;
        if (rl == 0) {
          p.save_mean[(long)g * p.C + c + j] = (float)m;
          p.save_invstd[(long)g * p.C + c + j] = (float)i;
          const double vu = (p.bessel && p.Mt > 1) ? var * p.Mt / (p.Mt - 1) : var;
          m0[j] -= (m0[j] - (float)m) * (1.f - p.decay);
          v0[j] -= (v0[j] - (float)vu) * (1.f - p.decay);
        }
      }
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int r = rl + i * R;
      if (r >= p.Mg) break;
      const long row = base + r;
      d4 u;
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = on ? fma((double)v[i][j] - mu[j], is[j], bt[j]) : 0.0;
      f4 y;
      int packed;
      float s;
      tape_row<L>(u, y, packed, s);
      if (on) {
        tde_st(reinterpret_cast<f4*>(p.y + row * p.ycs + p.yco + c), y);
        *reinterpret_cast<int*>(p.codes + row * p.C + c) = packed;
        if (l == 0) p.scales[row * p.NB + b] = s;
      }
    }
    // (the next group's first barrier orders its writes of sh after this group's reads; tot is rewritten only after it)
  }
  if (on && rl == 0 && p.mm)
#pragma unroll
    for (int j = 0; j < 4; ++j) { p.mm[c + j] = m0[j]; p.mv[c + j] = v0[j]; }
}

// ---- restore: the tape's values into channel views, one job per layer.  A row is C / 4 lanes, 256 / (C / 4) rows a step,
// eight rows in flight per lane (1572864 x 16: 21.8 us, 6.1 TB/s).
struct TapeRestore {
  tde_tape8_restore_t job[TDE_TAPE8_MULTI_MAX];
  int first[TDE_TAPE8_MULTI_MAX + 1];      // blocks of the jobs before this one
  int rpb[TDE_TAPE8_MULTI_MAX];            // rows per block
  int n, relu;
};

__global__ void __launch_bounds__(256) tape_restore_kernel(const TapeRestore p) {
  int k = 0;
  while (k + 1 < p.n && (int)blockIdx.x >= p.first[k + 1]) ++k;
  const tde_tape8_restore_t jb = p.job[k];
  const int nl = jb.C / 4, R = 256 / nl, NB = (jb.C + TDE_TAPE8_BLOCK - 1) / TDE_TAPE8_BLOCK;
  const int rl = threadIdx.x / nl, q = threadIdx.x - rl * nl, c = 4 * q, b = c / TDE_TAPE8_BLOCK;
  if (rl >= R) return;
  const long r0 = (long)(blockIdx.x - p.first[k]) * p.rpb[k], r1 = min((long)jb.M, r0 + p.rpb[k]);
  for (long rb = r0 + rl; rb < r1; rb += 8 * R) {
    int cd[8];
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long r = min(rb + i * R, r1 - 1);
      cd[i] = *reinterpret_cast<const int*>(jb.codes + r * jb.C + c);
      s[i] = jb.scales[r * NB + b];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long r = rb + i * R;
      if (r >= r1) break;
      f4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = tape_value(cd[i], j, s[i]);
        o[j] = p.relu && v < 0.f ? 0.f : v;
      }
      tde_st(reinterpret_cast<f4*>(jb.y + r * jb.y_cstride + jb.y_coff + c), o);
    }
  }
}

// ---- backward
struct TapeBwd {
  int Mg, C, NB, G;
  const int8_t* codes;
  const float *scales, *save_invstd, *beta, *dy;
  int dycs, dyco;
  double invM;               // 1 / rows per group over all replicas
  float *dz, *dbeta, *absmax;
  int acc;
};

__device__ __forceinline__ void tape_dz_row(const f4& dy, int q, float s, const f4& bt, const f4& m0, const f4& m1,
                                            const f4& is, f4& o, float& mx) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float xh = tape_value(q, j, s) - bt[j];
    const float g = (int8_t)(q >> (8 * j)) >= 0 ? dy[j] : 0.f;
    o[j] = is[j] * (g - m0[j] - xh * m1[j]);
    mx = fmaxf(mx, fabsf(o[j]));
  }
}

// (393216 x 32, dy of 68 channels: 24 us; 26565 x 36: 4.7)
template <int L>
__global__ void __launch_bounds__(256) tape_bwd_apply_kernel(const TapeBwd p, const double* gsums, const double* lsums,
                                                             int rpb) {
  const int nl = p.NB * L, R = 256 / nl;
  const int rl = threadIdx.x / nl, q = threadIdx.x - rl * nl, b = q / L, c = 4 * q, g = blockIdx.y;
  float mx = 0.f;
  if (rl < R && c < p.C) {
    const long base = (long)g * p.Mg;
    const int r0 = blockIdx.x * rpb, r1 = min(p.Mg, r0 + rpb);
    // (row addresses as in the forward)
    const unsigned zo = rl * p.C + c, so = rl * p.NB + b;
    const long yo = (long)rl * p.dycs + c;
    f4 v[APPLY_RB];
    int cd[APPLY_RB];
    float s[APPLY_RB];
    auto load = [&](int rb) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < APPLY_RB; ++i)
        if (rb + i * R + rl < r1) {
          const long row = base + rb + i * R;
          v[i] = *reinterpret_cast<const f4*>(p.dy + row * p.dycs + p.dyco + yo);
          cd[i] = *reinterpret_cast<const int*>(p.codes + row * p.C + zo);
          s[i] = p.scales[row * p.NB + so];
        }
    };
    load(r0);                          // in flight while the means are evaluated
    f4 m0, m1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m0[j] = (float)(gsums[(long)g * 2 * p.C + c + j] * p.invM);
      m1[j] = (float)(gsums[(long)g * 2 * p.C + p.C + c + j] * p.invM);
    }
    if (p.dbeta && blockIdx.x == 0 && g == 0 && rl == 0)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float db = p.acc ? p.dbeta[c + j] : 0.f;
        for (int gg = 0; gg < p.G; ++gg) db += (float)lsums[(long)gg * 2 * p.C + c + j];
        p.dbeta[c + j] = db;
      }
    const f4 is = *reinterpret_cast<const f4*>(p.save_invstd + (long)g * p.C + c);
    const f4 bt = *reinterpret_cast<const f4*>(p.beta + c);
    for (int rb = r0; rb < r1; rb += APPLY_RB * R) {
      f4 o[APPLY_RB];
#pragma unroll
      for (int i = 0; i < APPLY_RB; ++i)
        if (rb + i * R + rl < r1) tape_dz_row(v[i], cd[i], s[i], bt, m0, m1, is, o[i], mx);
      if (rb + APPLY_RB * R < r1) load(rb + APPLY_RB * R);
#pragma unroll
      for (int i = 0; i < APPLY_RB; ++i)
        if (rb + i * R + rl < r1) tde_st(reinterpret_cast<f4*>(p.dz + (base + rb + i * R) * p.C + zo), o[i]);
    }
  }
  block_absmax_to(mx, p.absmax);
}

template <int L, int RB>
__global__ void __launch_bounds__(SMALL_NT) tape_bwd_small_kernel(const TapeBwd p) {
  constexpr int R = SMALL_NT / L, NW = SMALL_NT / 64;
  __shared__ double sh[NW][L][8];
  __shared__ double tot[L][8];
  const int tid = threadIdx.x, l = tid % L, rl = tid / L, b = blockIdx.x, lane = tid & 63, wv = tid >> 6;
  const int c = 64 * b + 4 * l;
  const bool on = c < p.C;
  f4 bt = {0, 0, 0, 0};
  float db[4] = {0, 0, 0, 0}, mx = 0.f;
  if (on) {
    bt = *reinterpret_cast<const f4*>(p.beta + c);
    if (p.dbeta && p.acc && rl == 0)
#pragma unroll
      for (int j = 0; j < 4; ++j) db[j] = p.dbeta[c + j];
  }
  for (int g = 0; g < p.G; ++g) {
    const long base = (long)g * p.Mg;
    f4 v[RB];
    int cd[RB];
    float sc[RB];
    d4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int r = rl + i * R;
      const long row = base + r;
      const bool ok = on && r < p.Mg;
      v[i] = ok ? *reinterpret_cast<const f4*>(p.dy + row * p.dycs + p.dyco + c) : f4{0.f, 0.f, 0.f, 0.f};
      cd[i] = ok ? *reinterpret_cast<const int*>(p.codes + row * p.C + c) : -1;
      sc[i] = ok ? p.scales[row * p.NB + b] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      if (!on || rl + i * R >= p.Mg) break;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double xh = (double)(tape_value(cd[i], j, sc[i]) - bt[j]);
        const double gd = (int8_t)(cd[i] >> (8 * j)) >= 0 ? (double)v[i][j] : 0.0;
        s0[j] += gd;
        s1[j] = fma(gd, xh, s1[j]);
      }
    }
#pragma unroll
    for (int o = L; o < 64; o <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s0[j] += __shfl_xor(s0[j], o, 64);
        s1[j] += __shfl_xor(s1[j], o, 64);
      }
    if (lane < L)
#pragma unroll
      for (int j = 0; j < 4; ++j) { sh[wv][l][j] = s0[j]; sh[wv][l][4 + j] = s1[j]; }
    __syncthreads();
    if (tid < 8 * L) {
      double s = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) s += sh[w][tid >> 3][tid & 7];
      tot[tid >> 3][tid & 7] = s;
    }
    __syncthreads();
    if (on) {
      f4 m0, m1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m0[j] = (float)(tot[l][j] * p.invM);
        m1[j] = (float)(tot[l][4 + j] * p.invM);
        db[j] += (float)tot[l][j];
      }
      const f4 is = *reinterpret_cast<const f4*>(p.save_invstd + (long)g * p.C + c);
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const int r = rl + i * R;
        if (r >= p.Mg) break;
        f4 o;
        tape_dz_row(v[i], cd[i], sc[i], bt, m0, m1, is, o, mx);
        tde_st(reinterpret_cast<f4*>(p.dz + (base + r) * p.C + c), o);
      }
    }
  }
  if (on && rl == 0 && p.dbeta)
#pragma unroll
    for (int j = 0; j < 4; ++j) p.dbeta[c + j] = db[j];
  block_absmax_to(mx, p.absmax);
}

// ---- plans
constexpr int MAX_CHUNKS = 1024;   // row chunks of the sums over all groups and channel blocks (4 blocks per CU)

struct TapePlan {
  int L, NB, per_g, rpc;
};
TapePlan tape_plan(int M, int C, int G) {
  TapePlan t;
  t.L = tape_lanes(C);
  t.NB = (C + TDE_TAPE8_BLOCK - 1) / TDE_TAPE8_BLOCK;
  const int Mg = M / G, R = 256 / t.L;
  const long want = ((long)M * t.NB + MAX_CHUNKS - 1) / MAX_CHUNKS;      // rows of a chunk that fill MAX_CHUNKS blocks
  t.rpc = (int)(want > SUM_RB * R ? want : SUM_RB * R);
  t.per_g = tde_cdiv(Mg, t.rpc);
  return t;
}
// rows of an apply block: four steps of its row lanes, more when that is over 2048 blocks
int tape_apply_rows(int M, int C, const TapePlan& t) {
  const int R = 256 / (t.NB * t.L);
  const long want = ((long)M + 2047) / 2048;
  return (int)(want > 4 * R ? want : 4 * R);
}
bool tape_small(int Mg, int L) { return Mg <= SMALL_RB * SMALL_NT / L; }

#define TAPE_L(L, F)                 \
  switch (L) {                       \
    case 1: F(1); break;             \
    case 2: F(2); break;             \
    case 4: F(4); break;             \
    case 8: F(8); break;             \
    default: F(16); break;           \
  }

void tape_sums_launch(int mode, const TapePlan& t, int G, TapeSums p, double* part, double* sums, double* copy,
                      hipStream_t st) {
  p.NB = t.NB; p.per_g = t.per_g; p.rpc = t.rpc; p.part = part;
  const dim3 grid(G * t.per_g, t.NB);
#define F(LL)                                                                                          \
  if (mode == 0) hipLaunchKernelGGL((tape_sums_kernel<LL, 0>), grid, dim3(256), 0, st, p);             \
  else hipLaunchKernelGGL((tape_sums_kernel<LL, 1>), grid, dim3(256), 0, st, p)
  TAPE_L(t.L, F)
#undef F
  hipLaunchKernelGGL(tape_finalize_kernel, dim3(tde_cdiv(2 * p.C, 8), G), dim3(1024), 0, st, 2 * p.C, t.per_g, part,
                     sums, copy);
}
void tape_fwd_apply_launch(const TapePlan& t, const TapeFwd& p, const double* sums, hipStream_t st) {
  const int rpb = tape_apply_rows(p.Mg * p.G, p.C, t);
  const dim3 grid(tde_cdiv(p.Mg, rpb), p.G);
#define F(LL) hipLaunchKernelGGL(tape_fwd_apply_kernel<LL>, grid, dim3(256), 0, st, p, sums, rpb)
  TAPE_L(t.L, F)
#undef F
}
void tape_bwd_apply_launch(const TapePlan& t, const TapeBwd& p, const double* gs, const double* ls, hipStream_t st) {
  const int rpb = tape_apply_rows(p.Mg * p.G, p.C, t);
  const dim3 grid(tde_cdiv(p.Mg, rpb), p.G);
#define F(LL) hipLaunchKernelGGL(tape_bwd_apply_kernel<LL>, grid, dim3(256), 0, st, p, gs, ls, rpb)
  TAPE_L(t.L, F)
#undef F
}

bool tape_shape_ok(int M, int C, int groups) {
  return M > 0 && M <= (1 << 30) && C > 0 && C % 4 == 0 && C <= 1024 && groups >= 1 && groups <= BN_MAX_GROUPS && M % groups == 0;
}
bool tape_view_ok(const float* v, int C, int cs, int co) {
  return v && tde_aligned16(v) && cs % 4 == 0 && co % 4 == 0 && co >= 0 && (long)co + C <= cs;
}
bool tape_ok(const int8_t* codes, const float* scales) {
  return codes && scales && tde_aligned16(codes) && tde_aligned16(scales);
}
size_t tape_part_bytes(int M, int C) {
  // the most chunks any group count can ask for: one ragged chunk more per group
  const TapePlan t = tape_plan(M, C, 1);
  return (size_t)(t.per_g + BN_MAX_GROUPS) * 2 * C * sizeof(double);
}

}  // namespace

extern "C" {

size_t tde_tape8_workspace_size(int M, int C) {
  if (!tape_shape_ok(M, C, 1)) return 0;
  return tape_part_bytes(M, C) + (size_t)BN_MAX_GROUPS * 2 * C * sizeof(double);
}

int tde_tape8_one_launch(int M, int C, int groups) {
  return tape_shape_ok(M, C, groups) && tape_small(M / groups, tape_lanes(C)) ? 1 : 0;
}

int tde_tape8_bn_fwd(int M, int C, int groups, const float* z, const float* beta, float eps, float decay, int bessel,
                     float* moving_mean, float* moving_var, float* save_mean, float* save_invstd, float* y,
                     int y_cstride, int y_coff, int8_t* codes, float* scales, void* ws, size_t ws_bytes, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(tape_shape_ok(M, C, groups) && z && tde_aligned16(z) && beta && save_mean && save_invstd &&
                tape_view_ok(y, C, y_cstride, y_coff) && tape_ok(codes, scales) &&
                (moving_mean == nullptr) == (moving_var == nullptr));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const TapePlan t = tape_plan(M, C, groups);
  const TapeFwd p{M / groups, C, t.NB, groups, z, beta, (double)(M / groups), 1.0 / (M / groups), eps, decay, bessel, moving_mean, moving_var,
                  save_mean, save_invstd, y, y_cstride, y_coff, codes, scales};
  if (tape_small(p.Mg, t.L)) {
#define F(LL)                                                                                                       \
  if (p.Mg <= 2 * SMALL_NT / LL)                                                                                    \
    hipLaunchKernelGGL((tape_fwd_small_kernel<LL, 2>), dim3(t.NB), dim3(SMALL_NT), 0, st, p);                       \
  else if (p.Mg <= 4 * SMALL_NT / LL)                                                                               \
    hipLaunchKernelGGL((tape_fwd_small_kernel<LL, 4>), dim3(t.NB), dim3(SMALL_NT), 0, st, p);                       \
  else                                                                                                              \
    hipLaunchKernelGGL((tape_fwd_small_kernel<LL, SMALL_RB>), dim3(t.NB), dim3(SMALL_NT), 0, st, p)
    TAPE_L(t.L, F)
#undef F
    return tde_launch_status();
  }
  if (ws_bytes < tde_tape8_workspace_size(M, C) || !ws || !tde_aligned16(ws)) return TDE_ERR_WORKSPACE;
  double* part = reinterpret_cast<double*>(tde_ws_body(ws));
  double* sums = reinterpret_cast<double*>(tde_ws_body(ws) + tape_part_bytes(M, C));
  TapeSums s{};
  s.C = C; s.Mg = p.Mg; s.z = z;
  tape_sums_launch(0, t, groups, s, part, sums, nullptr, st);
  tape_fwd_apply_launch(t, p, sums, st);
  return tde_launch_status();
}

int tde_tape8_bn_fwd_from_sums(int M, int C, int groups, long M_total, const float* z, const double* sums,
                               const float* beta, float eps, float decay, int bessel, float* moving_mean,
                               float* moving_var, float* save_mean, float* save_invstd, float* y, int y_cstride,
                               int y_coff, int8_t* codes, float* scales, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(tape_shape_ok(M, C, groups) && M_total >= M / groups && z && tde_aligned16(z) && sums && beta &&
                save_mean && save_invstd && tape_view_ok(y, C, y_cstride, y_coff) && tape_ok(codes, scales) &&
                (moving_mean == nullptr) == (moving_var == nullptr));
  const TapePlan t = tape_plan(M, C, groups);
  const TapeFwd p{M / groups, C, t.NB, groups, z, beta, (double)M_total, 1.0 / (double)M_total, eps, decay, bessel, moving_mean, moving_var,
                  save_mean, save_invstd, y, y_cstride, y_coff, codes, scales};
  tape_fwd_apply_launch(t, p, sums, static_cast<hipStream_t>(stream));
  return tde_launch_status();
}

int tde_tape8_restore_multi(const tde_tape8_restore_t* jobs, int n, int relu, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(jobs && n > 0 && n <= TDE_TAPE8_MULTI_MAX && (relu == 0 || relu == 1));
  TapeRestore p{};
  p.n = n; p.relu = relu;
  for (int k = 0; k < n; ++k) {
    const tde_tape8_restore_t& j = jobs[k];
    TDE_CHECK_ARG(tape_shape_ok(j.M, j.C, 1) && tape_ok(j.codes, j.scales) && tape_view_ok(j.y, j.C, j.y_cstride, j.y_coff));
    p.job[k] = j;
    const int R = 256 / (j.C / 4);
    const long want = ((long)j.M + 2047) / 2048;      // at most 2048 blocks a job, eight steps of its row lanes each
    p.rpb[k] = (int)(want > 8 * R ? want : 8 * R);
    p.first[k + 1] = p.first[k] + tde_cdiv(j.M, p.rpb[k]);
  }
  hipLaunchKernelGGL(tape_restore_kernel, dim3(p.first[n]), dim3(256), 0, static_cast<hipStream_t>(stream), p);
  return tde_launch_status();
}

int tde_tape8_restore(int M, int C, const int8_t* codes, const float* scales, int relu, float* y, int y_cstride,
                      int y_coff, void* stream) {
  const tde_tape8_restore_t job{M, C, codes, scales, y, y_cstride, y_coff};
  return tde_tape8_restore_multi(&job, 1, relu, stream);
}

int tde_tape8_bn_bwd_sums(int M, int C, int groups, const int8_t* codes, const float* scales, const float* beta,
                          const float* dy, int dy_cstride, int dy_coff, double* sums, double* sums_copy, void* ws,
                          size_t ws_bytes, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(tape_shape_ok(M, C, groups) && tape_ok(codes, scales) && beta && tde_aligned16(beta) &&
                tape_view_ok(dy, C, dy_cstride, dy_coff) && sums);
  if (ws_bytes < tde_tape8_workspace_size(M, C) || !ws || !tde_aligned16(ws)) return TDE_ERR_WORKSPACE;
  TapeSums s{};
  s.C = C; s.Mg = M / groups; s.codes = codes; s.scales = scales; s.beta = beta; s.dy = dy; s.dycs = dy_cstride;
  s.dyco = dy_coff;
  tape_sums_launch(1, tape_plan(M, C, groups), groups, s, reinterpret_cast<double*>(tde_ws_body(ws)), sums, sums_copy,
                   static_cast<hipStream_t>(stream));
  return tde_launch_status();
}

int tde_tape8_bn_bwd_from_sums(int M, int C, int groups, long M_total, const int8_t* codes, const float* scales,
                               const float* save_invstd, const float* beta, const float* dy, int dy_cstride,
                               int dy_coff, const double* global_sums, const double* local_sums, float* dz,
                               float* dbeta, int accumulate_dbeta, float* dz_absmax, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(tape_shape_ok(M, C, groups) && M_total >= M / groups && tape_ok(codes, scales) && save_invstd && beta &&
                tde_aligned16(save_invstd) && tde_aligned16(beta) && tape_view_ok(dy, C, dy_cstride, dy_coff) &&
                global_sums && local_sums && dz && tde_aligned16(dz));
  const TapePlan t = tape_plan(M, C, groups);
  const TapeBwd p{M / groups, C, t.NB, groups, codes, scales, save_invstd, beta, dy, dy_cstride, dy_coff,
                  1.0 / (double)M_total, dz, dbeta, dz_absmax, accumulate_dbeta};
  tape_bwd_apply_launch(t, p, global_sums, local_sums, static_cast<hipStream_t>(stream));
  return tde_launch_status();
}

int tde_tape8_bn_bwd(int M, int C, int groups, const int8_t* codes, const float* scales, const float* save_invstd,
                     const float* beta, const float* dy, int dy_cstride, int dy_coff, float* dz, float* dbeta,
                     int accumulate_dbeta, float* dz_absmax, void* ws, size_t ws_bytes, void* stream) {
  tde_clear_error();
  TDE_CHECK_ARG(tape_shape_ok(M, C, groups) && tape_ok(codes, scales) && save_invstd && beta &&
                tde_aligned16(save_invstd) && tde_aligned16(beta) && tape_view_ok(dy, C, dy_cstride, dy_coff) && dz &&
                tde_aligned16(dz));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const TapePlan t = tape_plan(M, C, groups);
  const TapeBwd p{M / groups, C, t.NB, groups, codes, scales, save_invstd, beta, dy, dy_cstride, dy_coff,
                  1.0 / (double)(M / groups), dz, dbeta, dz_absmax, accumulate_dbeta};
  if (tape_small(p.Mg, t.L)) {
#define F(LL)                                                                                                       \
  if (p.Mg <= 2 * SMALL_NT / LL)                                                                                    \
    hipLaunchKernelGGL((tape_bwd_small_kernel<LL, 2>), dim3(t.NB), dim3(SMALL_NT), 0, st, p);                       \
  else if (p.Mg <= 4 * SMALL_NT / LL)                                                                               \
    hipLaunchKernelGGL((tape_bwd_small_kernel<LL, 4>), dim3(t.NB), dim3(SMALL_NT), 0, st, p);                       \
  else                                                                                                              \
    hipLaunchKernelGGL((tape_bwd_small_kernel<LL, SMALL_RB>), dim3(t.NB), dim3(SMALL_NT), 0, st, p)
    TAPE_L(t.L, F)
#undef F
    return tde_launch_status();
  }
  if (ws_bytes < tde_tape8_workspace_size(M, C) || !ws || !tde_aligned16(ws)) return TDE_ERR_WORKSPACE;
  double* part = reinterpret_cast<double*>(tde_ws_body(ws));
  double* sums = reinterpret_cast<double*>(tde_ws_body(ws) + tape_part_bytes(M, C));
  TapeSums s{};
  s.C = C; s.Mg = p.Mg; s.codes = codes; s.scales = scales; s.beta = beta; s.dy = dy; s.dycs = dy_cstride;
  s.dyco = dy_coff;
  tape_sums_launch(1, t, groups, s, part, sums, nullptr, st);
  tape_bwd_apply_launch(t, p, sums, sums, st);
  return tde_launch_status();
}

}  // extern "C"
