// Group normalisation + activation over channels-last activations [N][HW][C] for gfx950: per image n and group
// g of C/G neighbouring channels, over the m = HW * C/G values of the group,
//
//   forward    mean, rstd = 1 / sqrt(var + eps);  xhat = (x - mean) * rstd;  y = act(xhat * gamma + beta)
//   backward   dz = dy * act'(z);  dbeta = sum_{n,hw} dz;  dgamma = sum_{n,hw} dz * xhat
//              dx = rstd * (gamma*dz - m1 - xhat*m2),  m1 = mean_group(gamma*dz),  m2 = mean_group(gamma*dz*xhat)
//
// x, y, dy, dx: bf16, f16 or f32; gamma, beta, statistics, a thread's sums, and the backward's sums over threads and over a
// group's channels: f32; one rounding, of the result.
// Statistics of an image never leave it, so nothing is shared between images but the gamma / beta gradients, which a last
// kernel sums in a fixed order (no atomics: results repeat bit for bit).
//
// Variance: every thread takes the mean c of a few values that it holds and M = sum of (x - c)^2 around it; sets of n values
// meet as  M = sum of M_t + n_t (c_t - mean)^2.  Nothing but squares is added, so neither a mean far from zero nor a value
// far from the others cancels: rstd is good to a few units of f32 whatever the data.  Between threads and pieces sets meet
// in f64 and in one pass, around the first set's c: M = sum of M_t + n_t d_t^2 - (sum of n_t d_t)^2 / n with d_t = c_t - c_0.
// What that cancels is n (c_0 - mean)^2 of at least n_0 (c_0 - mean)^2: n / n_0 units of f64's 2^-53.
// (Sums around one value of the group, its first: 5e-5 off where that value lies 30 standard deviations from the mean,
// 2e-3 at 300.  E[x^2] - mean^2 loses mean^2 / var * 6e-8.)
#include "dtp_common.h"

#include <utility>

namespace {

constexpr int GN_MAXC = 4096;        // channels: a block's per-channel sums live in LDS (2 * C floats)

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2 };

struct tag_bf16 { static constexpr int size = 2; };
struct tag_f16 { static constexpr int size = 2; };
struct tag_f32 { static constexpr int size = 4; };

// VEC values of one row as a machine word (2, 4, 8 or 16 bytes): one load, unpacked where it is used
template <int BYTES> struct Word;
template <> struct Word<2> { typedef uint16_t t; };
template <> struct Word<4> { typedef uint32_t t; };
template <> struct Word<8> { typedef u32x2_t t; };
template <> struct Word<16> { typedef u32x4_t t; };

template <class T, int VEC> struct Pack {
  typedef typename Word<T::size * VEC>::t word;
  DTP_DEVINL static uint32_t half_at(const word& w, int e) {
    if constexpr (VEC == 1) return w;
    else if constexpr (VEC == 2) return (w >> (16 * (e & 1))) & 0xFFFFu;
    else return (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
  }
  DTP_DEVINL static void unpack(const word& w, float* f) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (T::size == 4) {
        if constexpr (VEC == 1) f[e] = __uint_as_float(w);
        else f[e] = __uint_as_float(w[e]);
      } else if constexpr (__is_same(T, tag_bf16)) {
        f[e] = __uint_as_float(half_at(w, e) << 16);
      } else {
        f[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)half_at(w, e));
      }
    }
  }
  DTP_DEVINL static uint32_t bits16(float f) {
    if constexpr (__is_same(T, tag_bf16)) return f32_to_bf16(f);
    else return __builtin_bit_cast(uint16_t, (_Float16)f);
  }
  DTP_DEVINL static word pack(const float* f) {
    word w;
    if constexpr (T::size == 4) {
      if constexpr (VEC == 1) w = __float_as_uint(f[0]);
      else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] = __float_as_uint(f[e]);
      }
    } else if constexpr (VEC == 1) {
      w = (uint16_t)bits16(f[0]);
    } else if constexpr (VEC == 2) {
      w = bits16(f[0]) | (bits16(f[1]) << 16);
    } else {
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) {
        if constexpr (__is_same(T, tag_bf16)) w[e] = pack_bf16x2(f[2 * e], f[2 * e + 1]);
        else w[e] = bits16(f[2 * e]) | (bits16(f[2 * e + 1]) << 16);
      }
    }
    return w;
  }
};

// 1 / (1 + exp(-z)).  f32 data: the library's exp and an IEEE division.  16-bit data: the hardware's exp2 and reciprocal,
// forward 64x56x56x256 bf16 48 us instead of 75, backward 94 instead of 140.  The rounded exponent makes exp(-z) |z| 2^-24 off,
// exp2 and reciprocal 2^-23 each: the sigmoid is at most 2^-22 off (absolute: |z| s (1 - s) <= 0.23), 2^-12 of f16's step at
// 1 and 2^-15 of bf16's; dgamma and dbeta are sums, in f32, of terms that are off by so much.
template <class T> DTP_DEVINL float sigmoid(float z) {
  if constexpr (T::size == 4) return 1.f / (1.f + expf(-z));
  else return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}
template <class T, int ACT> DTP_DEVINL float act_fwd(float z) {
  if constexpr (ACT == ACT_RELU) return z <= 0.f ? 0.f : z;            // NaN stays NaN
  else if constexpr (ACT == ACT_SILU) return z * sigmoid<T>(z);
  else return z;
}
template <class T, int ACT> DTP_DEVINL float act_bwd(float z, float dy) {
  if constexpr (ACT == ACT_RELU) return z > 0.f ? dy : 0.f;
  else if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid<T>(z);
    return dy * s * (1.f + z * (1.f - s));
  } else return dy;
}
// f(activation), chosen once for all rows (a choice at every value: backward 64x28x28x512 53 us, now 43)
template <class F> DTP_DEVINL void with_act(int act, F&& f) {
  if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>{});
  else if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>{});
  else f(std::integral_constant<int, ACT_NONE>{});
}

template <int CTRL> DTP_DEVINL float add_turned(float v) {       // v + v of the lane that many places on in its row of 16
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL> DTP_DEVINL double add_turned(double v) {
  return v + __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, true),
                              __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, true));
}
DTP_DEVINL double wave_reduce_sum_f64(double v) {
  v = add_turned<0x121>(v);                          // row_ror:1, 2, 4, 8
  v = add_turned<0x122>(v);
  v = add_turned<0x124>(v);
  v = add_turned<0x128>(v);
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

DTP_DEVINL double not_negative(double v) { return v < 0.0 ? 0.0 : v; }      // NaN stays NaN

struct GnShape {
  int N, HW, C, G, cpg;      // cpg = C / G
  int CV;                    // C / VEC
  int chunks, rows;          // an image's rows in `chunks` pieces of `rows`
  int once;                  // so many pieces from the front are read past the caches (GN_KEEP)
};

// n rows dealt out in turn: how many the k-th of R threads gets
struct Deal {
  int each, more;
  DTP_DEVINL Deal(int n, int R) : each(n / R), more(n - n / R * R) {}
  DTP_DEVINL int operator()(int k) const { return each + (k < more ? 1 : 0); }
};

// ---------------------------------------------------------------------------------------------------------
// Images whose groups fit a workgroup's registers: x is read once and y written once (backward: x and dy read once).
// A workgroup owns a slab of whole groups of one image: HW rows of TX vectors.  Threads stand in R = NT / TX rows of TX
// columns, a thread keeps its column and at most KV of its rows.
// Bound by HBM where it is large (64x56x56x256 bf16 forward 42 us = 4.9 TB/s), by one workgroup's load, fold and store where
// it is small (4x28x28x512 forward 7.5 us, backward 12.1 of which gn_dparam_kernel 3); backward at 223 registers a lane holds
// one workgroup a CU, so loads of one do not run under the stores of another (64x28x28x512 43 us, 3.6 TB/s).
struct GnSlab {
  int SG, slabs;             // groups of a slab, slabs of an image
};

// Sums over the threads of a column, from lanes of one wave first where TX is a power of two up to 32: afterwards
// `rows` rows of sums are to be added, and this thread has one of them if the result is >= 0.
DTP_DEVINL int column_rows(int TX, int NT, int ty, int R, int& rows) {
  const int lane = threadIdx.x & 63;
  if ((TX & (TX - 1)) == 0 && TX <= 32) {
    rows = NT >> 6;
    return lane < TX ? (int)(threadIdx.x >> 6) : -1;
  }
  rows = R;
  return ty < R ? ty : -1;
}
DTP_DEVINL float column_sum(float v, int TX) {       // over the lanes l, l + TX, ... of the wave
  if ((TX & (TX - 1)) != 0 || TX > 32) return v;
  if (TX <= 1) v = add_turned<0x121>(v);             // row_ror:1, 2, 4, 8
  if (TX <= 2) v = add_turned<0x122>(v);
  if (TX <= 4) v = add_turned<0x124>(v);
  if (TX <= 8) v = add_turned<0x128>(v);
  if (TX <= 16) v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
// groups (within a slab) of VEC neighbouring channels from c
template <int VEC> DTP_DEVINL void groups_of(int c, int cpg, int* g) {
  int q = c / cpg, left = cpg - (c - q * cpg);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    g[e] = q;
    if (--left == 0) { ++q; left = cpg; }
  }
}

// Sums over the u neighbours that make a unit, left in each of them
template <int VEC> DTP_DEVINL void unit_sums(float* a, int u) {
  if constexpr (VEC > 1) {
    if (u >= 2) {
#pragma unroll
      for (int e = 0; e < VEC; e += 2) a[e] = a[e + 1] = a[e] + a[e + 1];
    }
  }
  if constexpr (VEC > 2) {
    if (u >= 4) {
#pragma unroll
      for (int e = 0; e < VEC; e += 4) a[e] = a[e + 1] = a[e + 2] = a[e + 3] = a[e] + a[e + 2];
    }
  }
  if constexpr (VEC > 4) {
    if (u >= 8) {
      const float t = a[0] + a[4];
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[e] = t;
    }
  }
}

// The unit's first value in each of its places
template <int VEC> DTP_DEVINL void unit_first(float* a, int u) {
#pragma unroll
  for (int e = 1; e < VEC; ++e)
    if ((e & (u - 1)) != 0) a[e] = a[e - 1];
}

// f(0), f(1), .. f(N - 1) with the number known where the body is compiled: as a loop, the kept words of some types came to
// lie in one wide vector, copied at every row's condition (up to 3.5 KB a lane in scratch memory).
template <class F, int... I> DTP_DEVINL void each_of(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F> DTP_DEVINL void each(F&& f) { each_of(f, std::make_integer_sequence<int, N>{}); }

template <class T, int VEC, int NT, int KV>
__global__ __launch_bounds__(NT) void gn_slab_fwd_kernel(const void* __restrict__ x_, const float* __restrict__ gamma,
                                                         const float* __restrict__ beta, void* __restrict__ y_,
                                                         float* __restrict__ stats, const GnShape s, const GnSlab sl,
                                                         const float eps, const int act) {
  typedef typename Pack<T, VEC>::word word;
  extern __shared__ float sm[];                     // [3][R][units of a row], then [SG][2] mean, rstd
  const int block = xcd_remap(blockIdx.x, gridDim.x);
  const int n = block / sl.slabs, slab = block - n * sl.slabs;
  const int g0 = slab * sl.SG, ng = min(sl.SG, s.G - g0);
  const int TX = ng * s.cpg / VEC, R = NT / TX;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int c0 = g0 * s.cpg + tx * VEC;             // first channel of this thread
  const size_t base = (size_t)n * s.HW * s.CV;
  const word* xn = (const word*)x_ + base + c0 / VEC;
  word w[KV];
  each<KV>([&](auto i) {
    const int r = ty + i * R;
    if (ty < R && r < s.HW) w[i] = xn[(size_t)r * s.CV];
  });
  // neighbouring channels of one group and thread are one unit of u = gcd(cpg, VEC)
  int u = 1;
  if (VEC > 1 && s.cpg % 2 == 0) u = 2;
  if (VEC > 2 && s.cpg % 4 == 0) u = 4;
  if (VEC > 4 && s.cpg % 8 == 0) u = 8;
  const Deal dealt(s.HW, R);
  const int count = ty < R ? dealt(ty) * u : 0;
  const float inv = count ? 1.f / (float)count : 0.f;
  // (from the unit's first value: equal values have exactly their own mean, and no sum leaves f32 where the mean does not)
  float first[VEC], c[VEC], a0[VEC], a1[VEC];
  if (count) {
    Pack<T, VEC>::unpack(w[0], first);
    unit_first<VEC>(first, u);
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    if (!count) first[e] = 0.f;
    c[e] = a0[e] = a1[e] = 0.f;
  }
  each<KV>([&](auto i) {
    const int r = ty + i * R;
    if (ty < R && r < s.HW) {
      float f[VEC];
      Pack<T, VEC>::unpack(w[i], f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) c[e] = fmaf(f[e] - first[e], inv, c[e]);
    }
  });
  unit_sums<VEC>(c, u);
#pragma unroll
  for (int e = 0; e < VEC; ++e) c[e] += first[e];   // the thread's mean, or next to it: a0 is what it misses
  each<KV>([&](auto i) {
    const int r = ty + i * R;
    if (ty < R && r < s.HW) {
      float f[VEC];
      Pack<T, VEC>::unpack(w[i], f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = f[e] - c[e];
        a0[e] += d;
        a1[e] = fmaf(d, d, a1[e]);
      }
    }
  });
  unit_sums<VEC>(a0, u);
  unit_sums<VEC>(a1, u);
  const int nu = VEC / u, m = s.cpg / u, row = TX * nu, plane = R * row;
  if (ty < R) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (e % u == 0) {
        const int j = ty * row + tx * nu + e / u;
        const float miss = a0[e] * inv;
        sm[j] = c[e];
        sm[plane + j] = miss;
        sm[2 * plane + j] = fmaf(-a0[e], miss, a1[e]);
      }
    }
  }
  __syncthreads();
  float* ms = sm + 3 * plane;
  const int lane = threadIdx.x & 63;
  const double mm = (double)s.HW * s.cpg;
  for (int g = threadIdx.x >> 6; g < ng; g += NT / 64) {
    const double first = (double)sm[g * m] + (double)sm[plane + g * m];
    double a = 0.0, v = 0.0;
    for (int i = lane; i < R * m; i += 64) {
      const int r = i / m, j = r * row + g * m + i - r * m;
      const double d = ((double)sm[j] + (double)sm[plane + j]) - first, nd = (double)(dealt(r) * u) * d;
      a += nd;
      v += fma(nd, d, (double)sm[2 * plane + j]);
    }
    a = wave_reduce_sum_f64(a) / mm;
    v = wave_reduce_sum_f64(v) / mm;
    if (lane == 0) {
      const double mean = first + a;
      const float rstd = (float)(1.0 / sqrt(not_negative(fma(-a, a, v)) + (double)eps));
      ms[2 * g] = (float)mean;
      ms[2 * g + 1] = rstd;
      float* o = stats + ((size_t)n * s.G + g0 + g) * 2;
      o[0] = (float)mean;
      o[1] = rstd;
    }
  }
  __syncthreads();
  float mu[VEC], rs[VEC], ga[VEC], be[VEC];
  int gl[VEC];                                      // group within the slab
  groups_of<VEC>(tx * VEC, s.cpg, gl);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    mu[e] = ms[2 * gl[e]];
    rs[e] = ms[2 * gl[e] + 1];
    ga[e] = gamma[c0 + e];
    be[e] = beta[c0 + e];
  }
  word* yn = (word*)y_ + base + c0 / VEC;
  with_act(act, [&](auto which) {
    constexpr int ACT = decltype(which)::value;
    each<KV>([&](auto i) {
      const int r = ty + i * R;
      if (ty < R && r < s.HW) {
        float f[VEC], o[VEC];
        Pack<T, VEC>::unpack(w[i], f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = act_fwd<T, ACT>(fmaf((f[e] - mu[e]) * rs[e], ga[e], be[e]));
        yn[(size_t)r * s.CV] = Pack<T, VEC>::pack(o);
      }
    });
  });
}

// sums: per-channel (sum dz, sum dz*xhat) of every image, [N][2][C], for gn_dparam_kernel
template <class T, int VEC, int NT, int KV>
__global__ __launch_bounds__(NT) void gn_slab_bwd_kernel(const void* __restrict__ x_, const void* __restrict__ dy_,
                                                         const float* __restrict__ gamma, const float* __restrict__ beta,
                                                         const float* __restrict__ stats, void* __restrict__ dx_,
                                                         float* __restrict__ sums, const GnShape s, const GnSlab sl,
                                                         const int act) {
  typedef typename Pack<T, VEC>::word word;
  extern __shared__ float sm[];                     // [2][rows][channels], [2][channels], [SG][2]
  const int block = xcd_remap(blockIdx.x, gridDim.x);
  const int n = block / sl.slabs, slab = block - n * sl.slabs;
  const int g0 = slab * sl.SG, ng = min(sl.SG, s.G - g0);
  const int SC = ng * s.cpg, TX = SC / VEC, R = NT / TX;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int c0 = g0 * s.cpg + tx * VEC;
  const size_t base = (size_t)n * s.HW * s.CV + c0 / VEC;
  const word *xn = (const word*)x_ + base, *dn = (const word*)dy_ + base;
  word wx[KV], wd[KV];
  each<KV>([&](auto i) {
    const int r = ty + i * R;
    if (ty < R && r < s.HW) {
      wx[i] = xn[(size_t)r * s.CV];
      wd[i] = dn[(size_t)r * s.CV];
    }
  });
  float mu[VEC], rs[VEC], ga[VEC], be[VEC], a0[VEC], a1[VEC];
  int gl[VEC];
  groups_of<VEC>(tx * VEC, s.cpg, gl);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const float* st = stats + ((size_t)n * s.G + g0 + gl[e]) * 2;
    mu[e] = st[0];
    rs[e] = st[1];
    ga[e] = gamma[c0 + e];
    be[e] = beta[c0 + e];
    a0[e] = a1[e] = 0.f;
  }
  with_act(act, [&](auto which) {
    constexpr int ACT = decltype(which)::value;
    each<KV>([&](auto i) {
      const int r = ty + i * R;
      if (ty < R && r < s.HW) {
        float f[VEC], d[VEC];
        Pack<T, VEC>::unpack(wx[i], f);
        Pack<T, VEC>::unpack(wd[i], d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = (f[e] - mu[e]) * rs[e];
          const float dz = act_bwd<T, ACT>(fmaf(xh, ga[e], be[e]), d[e]);
          a0[e] += dz;
          a1[e] = fmaf(dz, xh, a1[e]);
        }
      }
    });
  });
  int rows;
  const int mine = column_rows(TX, NT, ty, R, rows);
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const float b0 = column_sum(a0[e], TX), b1 = column_sum(a1[e], TX);
    if (mine >= 0) {
      sm[mine * SC + tx * VEC + e] = b0;
      sm[(rows + mine) * SC + tx * VEC + e] = b1;
    }
  }
  __syncthreads();
  float *chs = sm + 2 * rows * SC, *ms = chs + 2 * SC;
  for (int i = threadIdx.x; i < 2 * SC; i += NT) {
    const int which = i >= SC, c = i - which * SC;
    float t = 0.f;
    for (int r = 0; r < rows; ++r) t += sm[(which * rows + r) * SC + c];
    sums[((size_t)n * 2 + which) * s.C + g0 * s.cpg + c] = t;
    chs[i] = t * gamma[g0 * s.cpg + c];
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const float inv = 1.f / ((float)s.HW * (float)s.cpg);
  for (int g = threadIdx.x >> 6; g < ng; g += NT / 64) {
    float b0 = 0.f, b1 = 0.f;
    for (int c = lane; c < s.cpg; c += 64) {
      b0 += chs[g * s.cpg + c];
      b1 += chs[SC + g * s.cpg + c];
    }
    b0 = wave_reduce_sum(b0);
    b1 = wave_reduce_sum(b1);
    if (lane == 0) {
      ms[2 * g] = b0 * inv;
      ms[2 * g + 1] = b1 * inv;
    }
  }
  __syncthreads();
  float m1[VEC], m2[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    m1[e] = ms[2 * gl[e]];
    m2[e] = ms[2 * gl[e] + 1];
  }
  word* on = (word*)dx_ + base;
  with_act(act, [&](auto which) {
    constexpr int ACT = decltype(which)::value;
    each<KV>([&](auto i) {
      const int r = ty + i * R;
      if (ty < R && r < s.HW) {
        float f[VEC], d[VEC], o[VEC];
        Pack<T, VEC>::unpack(wx[i], f);
        Pack<T, VEC>::unpack(wd[i], d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = (f[e] - mu[e]) * rs[e];
          const float dz = act_bwd<T, ACT>(fmaf(xh, ga[e], be[e]), d[e]);
          o[e] = rs[e] * (fmaf(ga[e], dz, -m1[e]) - xh * m2[e]);
        }
        on[(size_t)r * s.CV] = Pack<T, VEC>::pack(o);
      }
    });
  });
}

// ---------------------------------------------------------------------------------------------------------
// Any size: partial sums over pieces of an image, a fold, and a second pass over the data.
// A block's threads stand in rows of min(C / VEC, 256) columns; a thread keeps its column, so its channels'
// parameters stay in registers.
// Bound by HBM and the last-level cache: 64x224x224x64 bf16 forward 75 + 5 + 128 us, 6.0 TB/s; backward 122 + 6 + 209.
constexpr int GN_T = 256;

// Both passes over data that does not stay in the caches as a whole: the first reads from the front and the second from the
// back; what lies before the last GN_KEEP bytes is read past the caches, so that those bytes are still in the 256 MB
// last-level cache when the second pass comes to them; its results are written past the caches too.  Measured (us; in
// order with plain loads and stores / from the back, results past the caches / and GN_KEEP 128, 224, 256, 320 MB): forward
// 64x224x224x64 (411 MB) 272 / 253 / 216, 203, 204, 236, 256x224x224x64 - / 950 / 885, 859, 853, 916; backward
// 64x112x112x128 (411 MB) 232 / 186 / 181, 175, 174, 184, 64x56x56x256 (206 MB, all kept) 104 / 92.  Both passes over as
// many images at a time as the cache holds cost more in launches than it gains: 1120 for the 950.
constexpr double GN_KEEP = 240.0 * (1 << 20);

template <bool ONCE, class W> DTP_DEVINL W load_word(const W* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(p);
  else return *p;
}

// Forward: a thread takes its rows in runs of eight: their mean, their squares around it, and both join what it has (the
// formula at the head).  All of it relative to the mean of its first run, so that a large common mean costs no bits.
constexpr int GN_RUN = 8;

// BWD 0: per group of the piece its mean (as hi + lo) and M, the sum of squares around it -> partial [N][chunks][G][3]
// BWD 1: per channel (sum dz, sum dz*xhat) -> partial [N][chunks][2][C]
template <class T, int VEC, int BWD>
__global__ __launch_bounds__(GN_T) void gn_partial_kernel(const void* __restrict__ x_, const void* __restrict__ dy_,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta,
                                                          const float* __restrict__ stats, float* __restrict__ partial,
                                                          const GnShape s, const int act) {
  typedef typename Pack<T, VEC>::word word;
  extern __shared__ float sm[];                     // [2 + (BWD == 0)][GN_T * VEC] the threads'; BWD 0: channels' means (f64), M
  float* thr = sm;
  double* chm = (double*)(sm + 3 * GN_T * VEC);
  float* chv = (float*)(chm + s.C);
  const int n = blockIdx.x / s.chunks, chunk = blockIdx.x - n * s.chunks;
  const int r0 = chunk * s.rows, r1 = min(s.HW, r0 + s.rows);
  const word* xn = (const word*)x_ + (size_t)n * s.HW * s.CV;
  const word* dn = BWD ? (const word*)dy_ + (size_t)n * s.HW * s.CV : nullptr;
  const int TX = min(s.CV, GN_T), R = GN_T / TX;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  for (int cb = 0; cb < s.CV; cb += TX) {
    const int cv = cb + tx;
    const bool on = ty < R && cv < s.CV;
    float p[VEC], a0[VEC], a1[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) p[e] = a0[e] = a1[e] = 0.f;
    if (on) {
      if constexpr (BWD) {
        float rs[VEC], ga[VEC], be[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int c = cv * VEC + e, g = c / s.cpg;
          p[e] = stats[((size_t)n * s.G + g) * 2];
          rs[e] = stats[((size_t)n * s.G + g) * 2 + 1];
          ga[e] = gamma[c];
          be[e] = beta[c];
        }
        const auto rows = [&](auto once, auto which) {
          constexpr bool ONCE = decltype(once)::value;
          constexpr int ACT = decltype(which)::value;
#pragma unroll 4
          for (int r = r0 + ty; r < r1; r += R) {
            float f[VEC], d[VEC];
            Pack<T, VEC>::unpack(load_word<ONCE>(xn + (size_t)r * s.CV + cv), f);
            Pack<T, VEC>::unpack(load_word<ONCE>(dn + (size_t)r * s.CV + cv), d);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float xh = (f[e] - p[e]) * rs[e];
              const float dz = act_bwd<T, ACT>(fmaf(xh, ga[e], be[e]), d[e]);
              a0[e] += dz;
              a1[e] = fmaf(dz, xh, a1[e]);
            }
          }
        };
        with_act(act, [&](auto which) {
          if ((int)blockIdx.x < s.once) rows(std::true_type{}, which);
          else rows(std::false_type{}, which);
        });
      } else {
        // p: mean of this thread's first run, a0: of all its values less that, a1: M
        const auto rows = [&](auto once) {
          constexpr bool ONCE = decltype(once)::value;
          int r = r0 + ty;
          float have = 0.f;
          for (; r1 - r > (GN_RUN - 1) * R; r += GN_RUN * R) {
            word w[GN_RUN];
#pragma unroll
            for (int k = 0; k < GN_RUN; ++k) w[k] = load_word<ONCE>(xn + (size_t)(r + k * R) * s.CV + cv);
            float f[GN_RUN][VEC];
#pragma unroll
            for (int k = 0; k < GN_RUN; ++k) Pack<T, VEC>::unpack(w[k], f[k]);
            if (have == 0.f) {
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                p[e] = 0.f;
#pragma unroll
                for (int k = 1; k < GN_RUN; ++k) p[e] = fmaf(f[k][e] - f[0][e], 1.f / GN_RUN, p[e]);
                p[e] += f[0][e];
              }
            }
            const float all = have + GN_RUN, part = GN_RUN / all, both = have * part;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              float c = 0.f, q = 0.f;
#pragma unroll
              for (int k = 0; k < GN_RUN; ++k) {
                f[k][e] -= p[e];
                c += f[k][e];
              }
              c *= 1.f / GN_RUN;
#pragma unroll
              for (int k = 0; k < GN_RUN; ++k) {
                const float d = f[k][e] - c;
                q = fmaf(d, d, q);
              }
              const float d = c - a0[e];
              a0[e] = fmaf(d, part, a0[e]);
              a1[e] += fmaf(d * d, both, q);
            }
            have = all;
          }
          for (; r < r1; r += R) {
            float f[VEC];
            Pack<T, VEC>::unpack(load_word<ONCE>(xn + (size_t)r * s.CV + cv), f);
            const float all = have + 1.f, part = 1.f / all, both = have * part;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              if (have == 0.f) p[e] = f[e];
              const float d = (f[e] - p[e]) - a0[e];
              a0[e] = fmaf(d, part, a0[e]);
              a1[e] = fmaf(d * d, both, a1[e]);
            }
            have = all;
          }
        };
        if ((int)blockIdx.x < s.once) rows(std::true_type{});
        else rows(std::false_type{});
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        thr[(ty * TX + tx) * VEC + e] = a0[e];
        thr[GN_T * VEC + (ty * TX + tx) * VEC + e] = a1[e];
        if (!BWD) thr[2 * GN_T * VEC + (ty * TX + tx) * VEC + e] = p[e];
      }
    }
    __syncthreads();
    if constexpr (BWD) {
      for (int i = threadIdx.x; i < 2 * TX * VEC; i += GN_T) {
        const int which = i / (TX * VEC), j = i - which * TX * VEC, c = cb * VEC + j;
        if (c < s.C) {
          float t = 0.f;
          for (int k = 0; k < R; ++k) t += thr[which * GN_T * VEC + k * TX * VEC + j];
          partial[(((size_t)n * s.chunks + chunk) * 2 + which) * s.C + c] = t;
        }
      }
    } else {
      // P neighbouring lanes a channel, where channels are fewer than threads
      int P = 1;
      while (P < 64 && 2 * P * TX * VEC <= GN_T) P *= 2;
      const int len = r1 - r0, q = threadIdx.x & (P - 1);
      const Deal dealt(len, R);
      for (int j = threadIdx.x / P; j - (int)threadIdx.x / P < TX * VEC; j += GN_T / P) {
        const int c = cb * VEC + j;
        const auto mean_of = [&](int k) { return (double)thr[2 * GN_T * VEC + k * TX * VEC + j] + (double)thr[k * TX * VEC + j]; };
        const bool mine = j < TX * VEC && c < s.C;
        const double first = mine ? mean_of(0) : 0.0;
        double a = 0.0, v = 0.0;
        if (mine) {
#pragma unroll 4
          for (int k = q; k < R; k += P) {
            const double d = mean_of(k) - first, nd = (double)dealt(k) * d;
            a += nd;
            v += fma(nd, d, (double)thr[GN_T * VEC + k * TX * VEC + j]);
          }
        }
        for (int off = 1; off < P; off *= 2) {
          a += __shfl_xor(a, off, 64);
          v += __shfl_xor(v, off, 64);
        }
        if (mine && q == 0) {
          chm[c] = first + a / (double)len;
          chv[c] = (float)not_negative(v - a * a / (double)len);
        }
      }
    }
    __syncthreads();
  }
  if (!BWD) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int g = wave; g < s.G; g += GN_T / 64) {
      const double first = chm[g * s.cpg], len = (double)(r1 - r0);
      double a = 0.0, v = 0.0;
      for (int c = lane; c < s.cpg; c += 64) {
        const double d = chm[g * s.cpg + c] - first;
        a += d;
        v += fma(len * d, d, (double)chv[g * s.cpg + c]);
      }
      a = wave_reduce_sum_f64(a);
      v = wave_reduce_sum_f64(v);
      if (lane == 0) {
        v = not_negative(v - len * a * a / (double)s.cpg);
        a = first + a / (double)s.cpg;
        float* o = partial + (((size_t)n * s.chunks + chunk) * s.G + g) * 3;
        o[0] = (float)a;
        o[1] = (float)(a - (double)(float)a);
        o[2] = (float)v;
      }
    }
  }
}

// mean and rstd of (image, group) from its pieces: one wave each
__global__ __launch_bounds__(256) void gn_stats_kernel(const float* __restrict__ partial, float* __restrict__ stats,
                                                       const GnShape s, const float eps) {
  const long idx = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (idx >= (long)s.N * s.G) return;
  const int n = (int)(idx / s.G), g = (int)(idx - (long)n * s.G);
  const float* pn = partial + ((size_t)n * s.chunks * s.G + g) * 3;
  const double first = (double)pn[0] + (double)pn[1];
  double a = 0.0, v = 0.0;
#pragma unroll 4
  for (int k = lane; k < s.chunks; k += 64) {
    const float* o = pn + (size_t)k * s.G * 3;
    const double d = ((double)o[0] + (double)o[1]) - first, nd = (double)min(s.rows, s.HW - k * s.rows) * d;
    a += nd;
    v += fma(nd * (double)s.cpg, d, (double)o[2]);
  }
  a = wave_reduce_sum_f64(a) / (double)s.HW;
  v = wave_reduce_sum_f64(v) / ((double)s.HW * s.cpg);
  if (lane == 0) {
    stats[idx * 2] = (float)(first + a);
    stats[idx * 2 + 1] = (float)(1.0 / sqrt(not_negative(fma(-a, a, v)) + (double)eps));
  }
}

// Backward: per image, fold the pieces to per-channel sums [N][2][C] and per-group (m1, m2) [N][G][2].  A thread adds
// every `parts`-th piece of one value, eight loads under way (one thread a value, one load at a time: 20 us for 64 images
// of 56x56x256 in 32 pieces).
constexpr int GN_FOLD = 1024;
__global__ __launch_bounds__(GN_FOLD) void gn_bwd_fold_kernel(const float* __restrict__ partial,
                                                              const float* __restrict__ gamma, float* __restrict__ sums,
                                                              float* __restrict__ coef, const GnShape s) {
  extern __shared__ float sm[];                     // [2][C]
  __shared__ double part[GN_FOLD];
  const int n = blockIdx.x, W = 2 * s.C;
  const float* pn = partial + (size_t)n * s.chunks * W;
  const int parts = W >= GN_FOLD ? 1 : GN_FOLD / W, cols = min(W, GN_FOLD);
  for (int i0 = 0; i0 < W; i0 += cols) {
    const int i = i0 + threadIdx.x % cols, q = threadIdx.x / cols;
    double t = 0.0;
    if (q < parts && i < W) {
      int k = q;
      for (; k + 7 * parts < s.chunks; k += 8 * parts) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = pn[(size_t)(k + e * parts) * W + i];
#pragma unroll
        for (int e = 0; e < 8; ++e) t += (double)v[e];
      }
      for (; k < s.chunks; k += parts) t += (double)pn[(size_t)k * W + i];
    }
    part[threadIdx.x] = t;
    __syncthreads();
    if (q == 0 && i < W) {
      for (int k = 1; k < parts; ++k) t += part[k * cols + threadIdx.x];
      sums[(size_t)n * W + i] = (float)t;
      sm[i] = (float)t * gamma[i >= s.C ? i - s.C : i];
    }
    __syncthreads();
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float inv = 1.f / ((float)s.HW * (float)s.cpg);
  for (int g = wave; g < s.G; g += GN_FOLD / 64) {
    float u = 0.f, v = 0.f;
    for (int c = lane; c < s.cpg; c += 64) {
      u += sm[g * s.cpg + c];
      v += sm[s.C + g * s.cpg + c];
    }
    u = wave_reduce_sum(u);
    v = wave_reduce_sum(v);
    if (lane == 0) {
      coef[((size_t)n * s.G + g) * 2] = u * inv;
      coef[((size_t)n * s.G + g) * 2 + 1] = v * inv;
    }
  }
}

// dgamma / dbeta: the images' channel sums [N][2][C], 16 channels a block of 256 threads, 16 strands of images a channel,
// summed in f64 in a fixed order; written, or added to what is there (beta_* = 1)
struct GnParams {
  const float* sums;
  void *dgamma, *dbeta;
  int N, C, out_fp32;
  float beta_g, beta_b;
};

DTP_DEVINL void param_sums(const GnParams& p, const int block) {
  __shared__ double red[2][16][16];
  const int ci = threadIdx.x & 15, part = threadIdx.x >> 4, c = block * 16 + ci, C = p.C;
  double a = 0.0, b = 0.0;
  if (c < C) {
    for (int n = part; n < p.N; n += 16) {
      a += (double)p.sums[((size_t)n * 2) * C + c];
      b += (double)p.sums[((size_t)n * 2 + 1) * C + c];
    }
  }
  red[0][part][ci] = a;
  red[1][part][ci] = b;
  __syncthreads();
  if (part != 0 || c >= C) return;
  a = b = 0.0;
  for (int k = 0; k < 16; ++k) { a += red[0][k][ci]; b += red[1][k][ci]; }
  if (p.out_fp32) {
    float* dg = (float*)p.dgamma; float* db = (float*)p.dbeta;
    dg[c] = (p.beta_g != 0.f ? p.beta_g * dg[c] : 0.f) + (float)b;
    db[c] = (p.beta_b != 0.f ? p.beta_b * db[c] : 0.f) + (float)a;
  } else {
    bf16_t* dg = (bf16_t*)p.dgamma; bf16_t* db = (bf16_t*)p.dbeta;
    dg[c] = f32_to_bf16((p.beta_g != 0.f ? p.beta_g * bf16_to_f32(dg[c]) : 0.f) + (float)b);
    db[c] = f32_to_bf16((p.beta_b != 0.f ? p.beta_b * bf16_to_f32(db[c]) : 0.f) + (float)a);
  }
}
__global__ __launch_bounds__(256) void gn_dparam_kernel(const GnParams p) { param_sums(p, blockIdx.x); }

// Second pass; backward: its first `lead` blocks fold the parameters' gradients (64x56x56x256 87 us; in a launch of
// their own 92)
template <class T, int VEC, int BWD>
__global__ __launch_bounds__(GN_T) void gn_apply_kernel(const void* __restrict__ x_, const void* __restrict__ dy_,
                                                        const float* __restrict__ gamma, const float* __restrict__ beta,
                                                        const float* __restrict__ stats, const float* __restrict__ coef,
                                                        void* __restrict__ out_, const GnShape s, const int act,
                                                        const int lead, const GnParams params) {
  typedef typename Pack<T, VEC>::word word;
  if (BWD && (int)blockIdx.x < lead) {
    param_sums(params, blockIdx.x);
    return;
  }
  const int block = gridDim.x - 1 - blockIdx.x;      // the pieces read last first
  const int n = block / s.chunks, chunk = block - n * s.chunks;
  const int r0 = chunk * s.rows, r1 = min(s.HW, r0 + s.rows);
  const size_t base = (size_t)n * s.HW * s.CV;
  const word* xn = (const word*)x_ + base;
  const word* dn = BWD ? (const word*)dy_ + base : nullptr;
  word* on = (word*)out_ + base;
  const int TX = min(s.CV, GN_T), R = GN_T / TX;
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  if (ty >= R) return;
  for (int cv = tx; cv < s.CV; cv += TX) {
    float mu[VEC], rs[VEC], ga[VEC], be[VEC], m1[VEC], m2[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = cv * VEC + e;
      const size_t gi = ((size_t)n * s.G + c / s.cpg) * 2;
      mu[e] = stats[gi];
      rs[e] = stats[gi + 1];
      ga[e] = gamma[c];
      be[e] = beta[c];
      if (BWD) { m1[e] = coef[gi]; m2[e] = coef[gi + 1]; }
    }
    const auto rows = [&](auto once, auto which) {
      constexpr bool ONCE = decltype(once)::value;
      constexpr int ACT = decltype(which)::value;
#pragma unroll 4
    for   (int r = r0 + ty; r < r1; r += R) {
        float f[VEC], o[VEC];
        Pack<T, VEC>::unpack(load_word<ONCE>(xn + (size_t)r * s.CV + cv), f);
        if (BWD) {
          float d[VEC];
          Pack<T, VEC>::unpack(load_word<ONCE>(dn + (size_t)r * s.CV + cv), d);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float xh = (f[e] - mu[e]) * rs[e];
            const float dz = act_bwd<T, ACT>(fmaf(xh, ga[e], be[e]), d[e]);
            o[e] = rs[e] * (fmaf(ga[e], dz, -m1[e]) - xh * m2[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[e] = act_fwd<T, ACT>(fmaf((f[e] - mu[e]) * rs[e], ga[e], be[e]));
        }
        __builtin_nontemporal_store(Pack<T, VEC>::pack(o), &on[(size_t)r * s.CV + cv]);
      }
    };
    with_act(act, [&](auto which) {
      if (block < s.once) rows(std::true_type{}, which);
      else rows(std::false_type{}, which);
    });
  }
}

// Pieces of an image: about 2,048 blocks in all (8 a CU), but no piece under 32 KB, where a block's fixed part
// (parameters, LDS fold) would outweigh its rows.
GnShape shape_of(int N, int HW, int C, int G, int vec, int elem, int bwd) {
  GnShape s;
  s.N = N; s.HW = HW; s.C = C; s.G = G; s.cpg = C / G; s.CV = C / vec;
  long want = (2048 + N - 1) / N;
  const long most = ((long)HW * C * elem + 32767) / 32768;
  if (want > most) want = most;
  if (want > HW) want = HW;
  if (want < 1) want = 1;
  s.rows = (int)((HW + want - 1) / want);
  s.chunks = (HW + s.rows - 1) / s.rows;
  const double all = (double)N * HW * C * elem * (1 + bwd);
  s.once = all <= GN_KEEP ? 0 : (int)((double)N * s.chunks * (1.0 - GN_KEEP / all));
  return s;
}

// (HW: kernels count rows in 32 bits, up to a piece's 2^20 rows past the end before they compare)
bool gn_ok(int N, int HW, int C, int G, int dtype, int act) {
  return N > 0 && HW > 0 && C > 0 && C <= GN_MAXC && G > 0 && C % G == 0 && dtype >= 0 && dtype <= 2 && act >= 0 &&
         act <= 2 && (long)HW < 0x80000000L - (1L << 21) && (long)HW * C < 0x7fffffffL && (long)N * HW < 0x7fffffffL;
}

// widest vector of at most 16 bytes that divides a row
int gn_vec(int C, int elem) {
  int v = 16 / elem;
  while (C % v) v >>= 1;
  return v;
}

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// LDS of a slab kernel (a slab may be the image's last, with fewer groups: any number of columns has its place)
size_t slab_lds(const GnShape& s, int vec, int sg, int nt, int bwd) {
  const size_t row = (size_t)nt * (bwd ? 2 * vec : 3 * (vec / gcd(s.cpg, vec)));
  return (row + (bwd ? (size_t)2 * sg * s.cpg : 0) + 2 * (size_t)sg) * sizeof(float);
}

// rows of a thread
long slab_rows(const GnShape& s, int vec, int sg, int nt) {
  const long tx = (long)sg * s.cpg / vec;
  return (s.HW + nt / tx - 1) / (nt / tx);
}

// Whether a slab of `sg` groups fits (columns, rows a thread, 64 KB of LDS): 0 no, else the threads
int slab_fits(const GnShape& s, int vec, int sg, int bwd) {
  static const int nt[3] = {256, 512, 1024}, kv[2][3] = {{8, 16, 14}, {8, 16, 0}};
  const long tx = (long)sg * s.cpg / vec;
  for (int v = 0; v < 3; ++v)
    if (kv[bwd][v] && tx <= nt[v] && slab_rows(s, vec, sg, nt[v]) <= kv[bwd][v] &&
        slab_lds(s, vec, sg, nt[v], bwd) <= 65536)
      return nt[v];
  return 0;
}

// Groups of a slab; 0: none fits, or its rows are so short (64 bytes, 32, 16) that the loads cost more than a second
// pass.  Rows should be whole cache lines, but every CU should have a workgroup (16x56x56x256 with 256 at least, rows of
// 32 bytes: forward 16 us, backward 26; with 512, rows of 16: 21 and 41).  Measured (us, slab / two passes; bf16 where
// nothing else stands, 32 groups): rows of 64 bytes and more always pay (forward 64x56x56x256 42 / 71, backward
// 64x28x28x512 43 / 54); of 32: forward 32x56x56x256 in f32 36 / 64, backward 32x56x56x256 46 / 52, but backward
// 64x56x56x256 119 / 89; of 16: forward 8x56x56x256 14 / 18, 16x112x112x128 38 / 45, but 64x112x112x128 196 / 112 and, on
// half of the CUs, 4x112x112x128 23 / 19; backward 8x56x56x256 22.5 / 23, but 16x80x80x256 66 / 55.
int slab_groups(const GnShape& s, int vec, int elem, int bwd, int& threads) {
  const int step = vec / gcd(s.cpg, vec);            // groups that make whole vectors
  const long total = (long)s.N * s.HW * s.C * elem;
  int best = 0;
  for (int sg = step; sg <= s.G; sg += step) {
    const int f = slab_fits(s, vec, sg, bwd);
    if (!f) break;
    const long blocks = (long)s.N * ((s.G + sg - 1) / sg), bytes = (long)sg * s.cpg * elem;
    if (best && (blocks < 256 || bytes > 128)) break;
    best = sg;
    threads = f;
    if (bytes >= 128) break;
  }
  if (!best || best == s.G) return best;
  const long bytes = (long)best * s.cpg * elem, blocks = (long)s.N * ((s.G + best - 1) / best);
  if (bytes < 32 && total > (8L << 20) && blocks < 256) return 0;
  if (bytes < 32 && total > ((bwd ? 16L : 56L) << 20)) return 0;
  if (bytes < 64 && bwd && total > (64L << 20)) return 0;
  return best;
}

// A launch holds fewer than 2^32 threads.
bool grids_fit(const GnShape& s, int vec, int elem, int bwd) {
  int nt;
  const int sg = slab_groups(s, vec, elem, bwd, nt);
  long most = sg ? (long)s.N * ((s.G + sg - 1) / sg) * nt : ((long)s.N * s.chunks + 256) * GN_T;
  if (!sg) most = max(most, bwd ? (long)s.N * GN_FOLD : ((long)s.N * s.G + 3) / 4 * 256);
  return most < 1L << 32;
}

size_t partial_floats(const GnShape& s, int bwd) {
  return bwd ? (size_t)s.N * s.chunks * 2 * s.C : (size_t)s.N * s.chunks * s.G * 3;
}

template <class T, int VEC>
int gn_run_fwd(const void* x, const float* gamma, const float* beta, void* y, float* stats, float* ws, size_t ws_floats,
               const GnShape& s, float eps, int act, hipStream_t st) {
  int NT = 0;
  GnSlab sl;
  sl.SG = slab_groups(s, VEC, T::size, 0, NT);
  if (sl.SG) {
    sl.slabs = (s.G + sl.SG - 1) / sl.SG;
    const size_t lds = slab_lds(s, VEC, sl.SG, NT, 0);
    const dim3 g((unsigned)((long)s.N * sl.slabs));
    if (NT == 256) hipLaunchKernelGGL((gn_slab_fwd_kernel<T, VEC, 256, 8>), g, dim3(256), lds, st, x, gamma, beta, y, stats, s, sl, eps, act);
    else if (NT == 512) hipLaunchKernelGGL((gn_slab_fwd_kernel<T, VEC, 512, 16>), g, dim3(512), lds, st, x, gamma, beta, y, stats, s, sl, eps, act);
    else hipLaunchKernelGGL((gn_slab_fwd_kernel<T, VEC, 1024, 14>), g, dim3(1024), lds, st, x, gamma, beta, y, stats, s, sl, eps, act);
    return DTP_CHECK_LAUNCH();
  }
  if (ws_floats < partial_floats(s, 0)) return -12;
  const size_t lds = (size_t)(3 * s.C + 3 * GN_T * VEC) * sizeof(float);
  if (lds > 65536 && hipFuncSetAttribute((const void*)gn_partial_kernel<T, VEC, 0>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)lds) != hipSuccess)
    return -2;
  const dim3 grid(s.N * s.chunks);
  hipLaunchKernelGGL((gn_partial_kernel<T, VEC, 0>), grid, dim3(GN_T), lds, st, x, nullptr, gamma, beta, nullptr, ws, s, act);
  hipLaunchKernelGGL(gn_stats_kernel, dim3((unsigned)(((long)s.N * s.G + 3) / 4)), dim3(256), 0, st, ws, stats, s, eps);
  hipLaunchKernelGGL((gn_apply_kernel<T, VEC, 0>), grid, dim3(GN_T), 0, st, x, nullptr, gamma, beta, stats, nullptr, y, s, act, 0, GnParams{});
  return DTP_CHECK_LAUNCH();
}

template <class T, int VEC>
int gn_run_bwd(const void* x, const void* dy, const float* gamma, const float* beta, const float* stats, void* dx,
               void* dgamma, void* dbeta, int out_fp32, float beta_g, float beta_b, float* ws, size_t ws_floats,
               const GnShape& s, int act, hipStream_t st) {
  const size_t np = partial_floats(s, 1), ns = (size_t)s.N * 2 * s.C, nc = (size_t)s.N * s.G * 2;
  if (ws_floats < ns) return -12;
  float *sums = ws, *coef = sums + ns, *partial = coef + nc;
  const int lead = (s.C + 15) / 16;
  const GnParams params = {sums, dgamma, dbeta, s.N, s.C, out_fp32, beta_g, beta_b};
  int NT = 0;
  GnSlab sl;
  sl.SG = slab_groups(s, VEC, T::size, 1, NT);
  if (sl.SG) {
    sl.slabs = (s.G + sl.SG - 1) / sl.SG;
    const size_t slds = slab_lds(s, VEC, sl.SG, NT, 1);
    const dim3 g((unsigned)((long)s.N * sl.slabs));
    if (NT == 256) hipLaunchKernelGGL((gn_slab_bwd_kernel<T, VEC, 256, 8>), g, dim3(256), slds, st, x, dy, gamma, beta, stats, dx, sums, s, sl, act);
    else hipLaunchKernelGGL((gn_slab_bwd_kernel<T, VEC, 512, 16>), g, dim3(512), slds, st, x, dy, gamma, beta, stats, dx, sums, s, sl, act);
    hipLaunchKernelGGL(gn_dparam_kernel, dim3(lead), dim3(256), 0, st, params);
    return DTP_CHECK_LAUNCH();
  }
  if (ws_floats < np + ns + nc) return -12;
  const size_t lds = (size_t)(2 * GN_T * VEC) * sizeof(float);
  const dim3 grid(s.N * s.chunks);
  hipLaunchKernelGGL((gn_partial_kernel<T, VEC, 1>), grid, dim3(GN_T), lds, st, x, dy, gamma, beta, stats, partial, s, act);
  hipLaunchKernelGGL(gn_bwd_fold_kernel, dim3(s.N), dim3(GN_FOLD), (size_t)2 * s.C * sizeof(float), st, partial, gamma, sums, coef, s);
  hipLaunchKernelGGL((gn_apply_kernel<T, VEC, 1>), dim3(grid.x + lead), dim3(GN_T), 0, st, x, dy, gamma, beta, stats, coef, dx, s, act,
                     lead, params);
  return DTP_CHECK_LAUNCH();
}

}  // namespace

#define GN_DISPATCH(FN, ...)                                      \
  do {                                                            \
    if (dtype == 2) {                                             \
      if (vec == 4) return FN<tag_f32, 4>(__VA_ARGS__);           \
      if (vec == 2) return FN<tag_f32, 2>(__VA_ARGS__);           \
      return FN<tag_f32, 1>(__VA_ARGS__);                         \
    }                                                             \
    if (dtype == 1) {                                             \
      if (vec == 8) return FN<tag_f16, 8>(__VA_ARGS__);           \
      if (vec == 4) return FN<tag_f16, 4>(__VA_ARGS__);           \
      if (vec == 2) return FN<tag_f16, 2>(__VA_ARGS__);           \
      return FN<tag_f16, 1>(__VA_ARGS__);                         \
    }                                                             \
    if (vec == 8) return FN<tag_bf16, 8>(__VA_ARGS__);            \
    if (vec == 4) return FN<tag_bf16, 4>(__VA_ARGS__);            \
    if (vec == 2) return FN<tag_bf16, 2>(__VA_ARGS__);            \
    return FN<tag_bf16, 1>(__VA_ARGS__);                          \
  } while (0)

// Floats of scratch that dtp_gn_fwd (bwd = 0) / dtp_gn_bwd (bwd = 1) need; (size_t)-1: shape refused.
extern "C" size_t dtp_gn_workspace(int N, int HW, int C, int G, int dtype, int bwd) {
  if (!gn_ok(N, HW, C, G, dtype, 0)) return (size_t)-1;
  const int elem = dtype == 2 ? 4 : 2, vec = gn_vec(C, elem);
  const GnShape s = shape_of(N, HW, C, G, vec, elem, bwd);
  if (!grids_fit(s, vec, elem, bwd)) return (size_t)-1;
  int nt;
  const size_t sums = bwd ? (size_t)N * 2 * C : 0;
  if (slab_groups(s, vec, elem, bwd, nt)) return sums;
  return sums + partial_floats(s, bwd) + (bwd ? (size_t)N * G * 2 : 0);
}

// x, y: [N][HW][C] (dtype 0 bf16, 1 f16, 2 f32), 16-byte aligned; gamma, beta: f32 [C]; stats: f32 [N][G][2] (mean, rstd)
extern "C" int dtp_gn_fwd(const void* x, const float* gamma, const float* beta, void* y, float* stats, float* ws,
                          size_t ws_floats, int N, int HW, int C, int G, int dtype, int act, float eps, hipStream_t st) {
  if (!gn_ok(N, HW, C, G, dtype, act)) return -10;
  const int elem = dtype == 2 ? 4 : 2, vec = gn_vec(C, elem);
  const GnShape s = shape_of(N, HW, C, G, vec, elem, 0);
  if (!grids_fit(s, vec, elem, 0)) return -10;
  GN_DISPATCH(gn_run_fwd, x, gamma, beta, y, stats, ws, ws_floats, s, eps, act, st);
}

// stats as dtp_gn_fwd left them; dgamma / dbeta: [C], f32 or bf16, written (beta_* = 0) or added to (beta_* = 1)
extern "C" int dtp_gn_bwd(const void* x, const void* dy, const float* gamma, const float* beta, const float* stats,
                          void* dx, void* dgamma, void* dbeta, int out_fp32, float beta_g, float beta_b, float* ws,
                          size_t ws_floats, int N, int HW, int C, int G, int dtype, int act, hipStream_t st) {
  if (!gn_ok(N, HW, C, G, dtype, act)) return -10;
  const int elem = dtype == 2 ? 4 : 2, vec = gn_vec(C, elem);
  const GnShape s = shape_of(N, HW, C, G, vec, elem, 1);
  if (!grids_fit(s, vec, elem, 1)) return -10;
  GN_DISPATCH(gn_run_bwd, x, dy, gamma, beta, stats, dx, dgamma, dbeta, out_fp32, beta_g, beta_b, ws, ws_floats, s, act, st);
}
