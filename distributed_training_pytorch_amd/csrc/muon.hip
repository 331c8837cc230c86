// Newton-Schulz orthogonalisation and the Muon update for gfx950.
//
// For a matrix G the iteration is X_0 = G / (|G|_F + eps), X_{k+1} = a X_k + b (X_k X_k^T) X_k + c (X_k X_k^T)^2 X_k;
// it drives every singular value of X_0 towards 1.  With m <= n the sides of G (a tall G is taken transposed):
// k steps after some X, X_k = Q_k X, and Q_k and A_k = X_k X_k^T are polynomials of A = X X^T: symmetric m x m
// matrices that all commute.  So a segment of steps touches the long side twice only:
//
//   A = X X^T;   per step  P = a I + b A + c A A;   Q <- P Q;   A <- P (P A);   at the segment's end  X <- Q X
//
// 3 m^2 n + (4 k - 3) m^3 operations for k steps, where products with a symmetric result count half, instead of
// k * (4 m^2 n + 2 m^3).
//
// Precision.  Q's eigenvalues span a^k (directions that X lacks) to about 1 (those it has): Q X cancels, and a
// rounding of Q counts a^k times.  Two choices follow.  Segments of at most three steps (5 = 3 + 2): a^3 = 41; one
// segment of five, a^5 = 484, is 1e-3 off for a matrix of rank one where a loop of f32 products is 8e-5 off, and
// 3 + 2 is 9e-5 off.  And every matrix is held as a pair of f16 values, hi + lo (22 bits), scaled by a power of
// two into f16's range; a product of two of them is three MFMA products, hi*hi + hi*lo + lo*hi, accumulated in f32
// (lo*lo is 2^-22 of the sum).  Single 16-bit values would be 1e-2 and more off.
//
// Layout of a [rows][K] matrix of pairs: in the matrix instruction's own order.  16 rows and 32 of K make a block of
// 2 KB: 64 lanes' 16 bytes of hi values (lane = row + 16 * (k / 8): values k..k+7 of the row), then the same of lo
// values; a row of blocks lies in the order of K.  A fragment is one contiguous kilobyte, from memory to registers,
// from memory to LDS and from LDS to registers, without bank conflicts and without a swizzle; with rows of K in memory a
// fragment touches 16 cache lines by half and a CU loads 16 bytes a clock instead of 64.
#include "dtp_common.h"

namespace {

typedef _Float16 f16_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4_t;
typedef __attribute__((ext_vector_type(4))) uint16_t u16x4_t;

constexpr int NS_MAXMAT = 24;            // matrices per call
constexpr int NS_PART = 1024;            // partial sums of squares per matrix
constexpr int NS_SPLIT = 8;              // workgroups that share a tile along K, where they do: one an XCD
constexpr int NS_SHARED = 64;            // most tiles of such a launch

// head of the workspace
constexpr long NS_AT_PART = 4096;                                              // sums of squares, f64
constexpr long NS_AT_SLABS = NS_AT_PART + (long)NS_MAXMAT * NS_PART * 8;         // shared tiles' sums
constexpr long NS_AT_MATS = NS_AT_SLABS + (long)NS_SHARED * NS_SPLIT * 64 * 64 * 4;

// workspace arrays of a matrix
enum { W_X = 0, W_XT0, W_XT1, W_A, W_P, W_R, W_Q0, W_Q1 };

struct NsMat {
  const void* src;        // G, or the gradient (muon)
  float* mom;             // muon: momentum, f32 [rows][cols]
  float* w;               // muon: weights, f32
  void* out;              // newton_schulz: result; muon: bf16 copy of the weights (may be null)
  int rows, cols;         // of G
  int m, n;               // padded sides, m <= n: multiples of 64
  long off[2];            // byte offsets into the workspace: [0] X, X^T, X^T in a row, [1] A, P, R, Q0, Q1
  float decay, step;      // muon: w = w * decay - step * O
  int aligned;            // src, mom, w, out start on 16 bytes
};

// The table travels as an argument of the first kernel, which leaves it at the head of the workspace: the other
// launches carry 200 bytes of arguments instead of 2 KB.
struct NsTable { NsMat mat[NS_MAXMAT]; };

struct NsBlocks {
  int first[NS_MAXMAT + 1];      // first block of each matrix in this launch
  int count;
  int shared;                    // tiles are shared out along K
};

DTP_DEVINL char* ws_at(char* ws, const NsMat& t, int which) {
  if (which <= W_XT1) return ws + t.off[0] + (long)which * t.m * t.n * 4;
  return ws + t.off[1] + (long)(which - W_A) * t.m * t.m * 4;
}

DTP_DEVINL int find_mat(const NsBlocks& tb, int block) {
  int i = 0;
  while (i + 1 < tb.count && block >= tb.first[i + 1]) ++i;
  return i;
}

__host__ __device__ inline int norm_blocks(int rows, int cols) {
  const long nb = ((long)rows * cols + 4095) / 4096;
  return nb > NS_PART ? NS_PART : (int)nb;
}

DTP_DEVINL void split_f16(float v, f16_t& hi, f16_t& lo) {
  hi = (f16_t)v;
  lo = (f16_t)(v - (float)hi);
}

constexpr int LO = 512;                  // lo values behind their hi values, in f16

// element (r, k) of a pair matrix of ld columns: offset of its hi value, in f16
DTP_DEVINL long pair_at(int r, int k, int ld) {
  return ((long)(r >> 4) * (ld >> 5) + (k >> 5)) * 1024 + (((r & 15) + 16 * ((k >> 3) & 3)) << 3) + (k & 7);
}

template <int KIND> DTP_DEVINL float load_as_f32(const void* p, long i) {   // 0 f32, 1 bf16, 2 f16
  if (KIND == 0) return ((const float*)p)[i];
  if (KIND == 1) return bf16_to_f32(((const bf16_t*)p)[i]);
  return (float)((const f16_t*)p)[i];
}

struct MuonArgs { float mu, omu, gscale; int nesterov; };      // omu = 1 - momentum

// momentum m <- mu*m + (1-mu)*grad; what is orthogonalised
DTP_DEVINL float muon_direction(float g, float& m, const MuonArgs& a) {
  g *= a.gscale;
  m = fmaf(a.omu, g, a.mu * m);
  return a.nesterov ? fmaf(a.mu, m, a.omu * g) : m;
}
// the same from the momentum already updated
DTP_DEVINL float muon_again(float g, float m, const MuonArgs& a) {
  return a.nesterov ? fmaf(a.mu, m, a.omu * (g * a.gscale)) : m;
}

DTP_DEVINL double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Sum of squares of G in f64 (any magnitude of G: no overflow, nothing lost on 10^8 values), one partial a block.
// Muon: momentum <- mu*momentum + (1-mu)*grad on the way; G = nesterov ? (1-mu)*grad + mu*momentum : momentum.
template <int KIND, int MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsTable tb, const NsBlocks bl, char* __restrict__ ws,
                                                      const MuonArgs ma) {
  __shared__ double red[4];
  double* part = (double*)(ws + NS_AT_PART);
  static_assert(sizeof(NsTable) <= NS_AT_PART, "the table's place");
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < bl.count * (int)(sizeof(NsMat) / 8); i += 256) ((long*)ws)[i] = ((const long*)tb.mat)[i];
  const int mi = find_mat(bl, blockIdx.x);
  const NsMat& t = tb.mat[mi];
  const int b = blockIdx.x - bl.first[mi], nb = bl.first[mi + 1] - bl.first[mi];
  const long total = (long)t.rows * t.cols, nvec = t.aligned ? total / 4 : 0;
  double s = 0.0;
#pragma unroll 4
  for (long i = (long)b * 256 + threadIdx.x; i < nvec; i += (long)nb * 256) {
    f32x4_t u;
    if (KIND == 0) {
      u = ((const f32x4_t*)t.src)[i];
    } else if (KIND == 1) {
      const u32x2_t q = ((const u32x2_t*)t.src)[i];
      u = (f32x4_t){__uint_as_float(q[0] << 16), __uint_as_float(q[0] & 0xFFFF0000u), __uint_as_float(q[1] << 16),
                    __uint_as_float(q[1] & 0xFFFF0000u)};
    } else {
      u = __builtin_convertvector(((const f16x4_t*)t.src)[i], f32x4_t);
    }
    if (MUON) {
      f32x4_t m = ((const f32x4_t*)t.mom)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float me = m[e];
        u[e] = muon_direction(u[e], me, ma);
        m[e] = me;
      }
      ((f32x4_t*)t.mom)[i] = m;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s += (double)u[e] * (double)u[e];
  }
  for (long i = nvec * 4 + (long)b * 256 + threadIdx.x; i < total; i += (long)nb * 256) {
    float u = load_as_f32<KIND>(t.src, i);
    if (MUON) {
      float m = t.mom[i];
      u = muon_direction(u, m, ma);
      t.mom[i] = m;
    }
    s += (double)u * (double)u;
  }
  s = wave_sum_f64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[mi * NS_PART + b] = red[0] + red[1] + red[2] + red[3];
}

// X_0 as pairs, in both orientations, zero-padded: one 64 x 64 tile of the padded matrix a block
template <int KIND, int MUON>
__global__ __launch_bounds__(256) void ns_split_kernel(const NsMat* __restrict__ mats, const NsBlocks bl,
                                                       char* __restrict__ ws, const double* __restrict__ part,
                                                       const MuonArgs ma, const float eps, const float scale) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int mi = find_mat(bl, blockIdx.x);
  const NsMat& t = mats[mi];
  const bool tall = t.rows > t.cols;
  const int pr = tall ? t.n : t.m, pc = tall ? t.m : t.n;          // padded rows / columns of G
  const int b = blockIdx.x - bl.first[mi], tc = pc / 64, br = b / tc, bc = b - br * tc;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float v[16];                                       // the loads of the tile and of the sums are under way together
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int gr = br * 64 + wave + 4 * i, gc = bc * 64 + lane;
    v[i] = 0.f;
    if (gr < t.rows && gc < t.cols) {
      const long at = (long)gr * t.cols + gc;
      v[i] = load_as_f32<KIND>(t.src, at);
      if (MUON) v[i] = muon_again(v[i], t.mom[at], ma);
    }
  }
  const int nparts = norm_blocks(t.rows, t.cols);
  double s = 0.0;
  for (int i = threadIdx.x; i < nparts; i += 256) s += part[mi * NS_PART + i];
  s = wave_sum_f64(s);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  const double inv = (double)scale / (sqrt(red[0] + red[1] + red[2] + red[3]) + (double)eps);
#pragma unroll
  for (int i = 0; i < 16; ++i) tile[wave + 4 * i][lane] = (float)((double)v[i] * inv);
  f16_t* same = (f16_t*)ws_at(ws, t, tall ? W_XT0 : W_X);
  f16_t* turn = (f16_t*)ws_at(ws, t, tall ? W_X : W_XT0);
  __syncthreads();
  // the tile is 4 x 2 blocks in either orientation; a wave writes one block at a time
  const int r = lane & 15, k = (lane >> 4) * 8;
#pragma unroll
  for (int q = wave; q < 16; q += 4) {
    const int rb = (q & 7) >> 1, kb = q & 1;
    const bool turned = q >= 8;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = turned ? tile[kb * 32 + k + e][rb * 16 + r] : tile[rb * 16 + r][kb * 32 + k + e];
    f16x8_t hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f16_t h, l;
      split_f16(x[e], h, l);
      hi[e] = h;
      lo[e] = l;
    }
    f16_t* to = turned ? turn + pair_at(bc * 64 + rb * 16 + r, br * 64 + kb * 32 + k, pr)
                       : same + pair_at(br * 64 + rb * 16 + r, bc * 64 + kb * 32 + k, pc);
    *(f16x8_t*)to = hi;
    *(f16x8_t*)(to + LO) = lo;
  }
}

// One product of pair matrices per matrix of the table: D = A B^T, both operands [rows][K] in pair layout.
struct NsOp { int a, b, d, dt; float scale; };       // operands, result, its transpose (-1: none), factor from the accumulator
struct NsGemm {
  NsOp op[2];
  int nops;
  int is_long;                                       // b is X^T: the result is m x n; otherwise it is m x m, symmetric
  int out_kind;                                      // EPI_OUT: 0 f32, 1 bf16, 2 f16, 3 muon
  float ca, cb;                                      // EPI_POLY: result = ca I + cb * A + scale * acc
};

enum { EPI_PAIR = 0, EPI_POLY = 1, EPI_OUT = 2 };

// Where a tile's product goes.
struct NsDest {
  const char* A;          // EPI_POLY: operand A
  char* D;                // result, [rows][cols] pairs
  char* DT;               // its transpose, or null
  int rows, cols;
  float scale;
};

// Four neighbouring values of O: the result, or the weights' update (out_kind 3: w = w * decay - step * O, in f32)
DTP_DEVINL void ns_out(const NsMat& t, const int out_kind, const int r, const int c, const f32x4_t v) {
  if (r >= t.rows || c >= t.cols) return;
  const long o = (long)r * t.cols + c;
  if ((t.cols & 3) == 0 && t.aligned) {
    if (out_kind == 0) *(f32x4_t*)((float*)t.out + o) = v;
    else if (out_kind == 1) *(u32x2_t*)((bf16_t*)t.out + o) = (u32x2_t){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    else if (out_kind == 2) *(f16x4_t*)((f16_t*)t.out + o) = __builtin_convertvector(v, f16x4_t);
    else {
      const f32x4_t w = *(const f32x4_t*)(t.w + o) * t.decay - v * t.step;
      *(f32x4_t*)(t.w + o) = w;
      if (t.out) *(u32x2_t*)((bf16_t*)t.out + o) = (u32x2_t){pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3])};
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (c + e >= t.cols) return;
    if (out_kind == 0) ((float*)t.out)[o + e] = v[e];
    else if (out_kind == 1) ((bf16_t*)t.out)[o + e] = f32_to_bf16(v[e]);
    else if (out_kind == 2) ((f16_t*)t.out)[o + e] = (f16_t)v[e];
    else {
      const float w = t.w[o + e] * t.decay - v[e] * t.step;
      t.w[o + e] = w;
      if (t.out) ((bf16_t*)t.out)[o + e] = f32_to_bf16(w);
    }
  }
}

// A wave stores 16 * MI rows from r0 and 16 * NI columns from c0: a lane holds row r0 + i*16 + (lane & 15), columns
// c0 + j*16 + (lane >> 4) * 4 + 0..3.  slab: 32 * (16 * NI + 2) words of LDS of the wave's own.
template <int MI, int NI, int EPI>
DTP_DEVINL void ns_store(const NsMat& t, const NsGemm& p, const NsDest& d, f32x4_t (&acc)[MI][NI], const int r0,
                         const int c0, uint32_t* slab) {
  constexpr int SLD = 16 * NI + 2;
  const int lane = threadIdx.x & 63, frow = lane & 15, fk = lane >> 4;
  if (EPI == EPI_OUT) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) ns_out(t, p.out_kind, r0 + i * 16 + frow, c0 + j * 16 + fk * 4, acc[i][j] * d.scale);
    return;
  }
  f16_t *D = (f16_t*)d.D, *DT = (f16_t*)d.DT;
#pragma unroll
  for (int ii = 0; ii < MI; ii += 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = ii + h, r = r0 + i * 16 + frow;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int c = c0 + j * 16 + fk * 4;
        f32x4_t v = acc[i][j] * d.scale;
        const bool in = r < d.rows && c < d.cols;
        const long o = pair_at(r, c, d.cols);
        if (EPI == EPI_POLY && in) {
          const f32x4_t ah = __builtin_convertvector(*(const f16x4_t*)((const f16_t*)d.A + o), f32x4_t);
          const f32x4_t al = __builtin_convertvector(*(const f16x4_t*)((const f16_t*)d.A + o + LO), f32x4_t);
          v += (ah + al) * p.cb;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e == r) v[e] += p.ca;
        }
        const f16x4_t hi = __builtin_convertvector(v, f16x4_t);
        const f16x4_t lo = __builtin_convertvector(v - __builtin_convertvector(hi, f32x4_t), f16x4_t);
        if (in) {
          *(f16x4_t*)(D + o) = hi;
          *(f16x4_t*)(D + o + LO) = lo;
        }
        if (DT) {
          const u16x4_t hb = __builtin_bit_cast(u16x4_t, hi), lb = __builtin_bit_cast(u16x4_t, lo);
          uint32_t* s = slab + (h * 16 + frow) * SLD + j * 16 + fk * 4;
          *(u32x2_t*)s = (u32x2_t){hb[0] | ((uint32_t)lb[0] << 16), hb[1] | ((uint32_t)lb[1] << 16)};
          *(u32x2_t*)(s + 2) = (u32x2_t){hb[2] | ((uint32_t)lb[2] << 16), hb[3] | ((uint32_t)lb[3] << 16)};
        }
      }
    }
    if (DT) {
      // 32 rows by 16 columns of the tile are one block of the transpose: a lane turns 8 rows of one column
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const int r = r0 + ii * 16;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int c = c0 + j * 16 + frow;
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = slab[(fk * 8 + e) * SLD + j * 16 + frow];
        if (c < d.cols && r < d.rows) {
          f16_t* to = DT + pair_at(c, r + fk * 8, d.rows);
          u32x4_t hi, lo;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            hi[e] = (w[2 * e] & 0xFFFFu) | (w[2 * e + 1] << 16);
            lo[e] = (w[2 * e] >> 16) | (w[2 * e + 1] & 0xFFFF0000u);
          }
          *(u32x4_t*)to = hi;
          *(u32x4_t*)(to + LO) = lo;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
}

// What a workgroup computes: matrix, operands, tile.
struct NsWork {
  int mat, m0, n0, K, split, nsplit;
  const char *A, *B;
  NsDest dest;
};

template <int BM, int BN, int EPI>
DTP_DEVINL NsWork ns_work(const NsMat* __restrict__ mats, const NsBlocks& tb, char* ws, const NsGemm& p, const int block) {
  NsWork w;
  w.mat = find_mat(tb, block);
  const NsMat& t = mats[w.mat];
  const bool tall = t.rows > t.cols;
  int b = block - tb.first[w.mat];
  w.nsplit = tb.shared ? NS_SPLIT : 1;
  w.split = b % w.nsplit;
  b /= w.nsplit;
  const int per = (tb.first[w.mat + 1] - tb.first[w.mat]) / w.nsplit / p.nops, oi = b / per;
  b -= oi * per;
  const NsOp op = p.op[oi];
  // EPI_OUT: O = Q X for a wide G, O = X^T Q for a tall one: rows and columns of O are G's
  const bool swap = EPI == EPI_OUT && tall;
  const int asel = swap ? op.b : op.a, bsel = swap ? op.a : op.b;
  const int rows = swap ? t.n : t.m, cols = swap || !p.is_long ? t.m : t.n;
  w.K = asel == W_X ? t.n : t.m;                     // the Gram product runs along the long side
  // Tiles in order of groups of four tile rows, down a group's columns: neighbours, which share an L2, form squares and
  // read few rows of blocks between them.  Symmetric results: on and below the diagonal (BM == BN).
  int ti, tj;
  const int tr = (rows + BM - 1) / BM, tc = (cols + BN - 1) / BN;
  if (!p.is_long) {
    int row = (int)((sqrtf(8.f * b + 1.f) - 1.f) * 0.5f);
    while (row * (row + 1) / 2 > b) --row;
    while ((row + 1) * (row + 2) / 2 <= b) ++row;
    const int r0 = row & ~3, h = min(4, tr - r0);
    int y = b - r0 * (r0 + 1) / 2;
    if (y < r0 * h) {
      ti = r0 + y % h;
      tj = y / h;
    } else {
      y -= r0 * h;
      int d = 0;
      while ((d + 1) * (d + 2) / 2 <= y) ++d;
      ti = r0 + d;
      tj = r0 + y - d * (d + 1) / 2;
    }
  } else {
    const int r0 = b / (4 * tc) * 4, h = min(4, tr - r0), y = b - r0 * tc;
    ti = r0 + y % h;
    tj = y / h;
  }
  w.m0 = ti * BM;
  w.n0 = tj * BN;
  w.A = ws_at(ws, t, asel);
  w.B = ws_at(ws, t, bsel);
  w.dest = {w.A, nullptr, nullptr, rows, cols, op.scale};
  if (EPI != EPI_OUT) {
    w.dest.D = ws_at(ws, t, op.d);
    w.dest.DT = p.is_long ? ws_at(ws, t, op.dt) : ti != tj ? w.dest.D : nullptr;
  }
  return w;
}

// Large tiles: a ring of NST stages of LDS-DMA with counted waits; a wave reads the next step's fragments into registers
// while it multiplies this one's, a read behind every two or three matrix instructions (4096 x 4096: 3.66 ms, with the
// reads in front of the products 3.90).  192 x 192 by eight waves, 128 x 128 by four.  Bound by the power the matrix
// pipes draw: 4096 x 25088 runs at 1.1 PFLOP/s, three products counted for each of the pairs', and a bare loop of this
// instruction on random values, no memory touched, sustains 1.65.  (256 x 256 was 20 % slower on 4096 x 4096: 136 tiles
// leave half the CUs idle where 192 x 192 has 253.  The 32x32x16 instruction with four waves: 13 % slower.)
template <int BM, int BN, int WGM, int WGN, int NST, int EPI>
__global__ __launch_bounds__(WGM * WGN * 64) void ns_gemm_kernel(const NsMat* __restrict__ mats, const NsBlocks tb, char* __restrict__ ws, const NsGemm p) {
  constexpr int T = WGM * WGN * 64;
  constexpr int WM = BM / WGM, WN = BN / WGN, MI = WM / 16, NI = WN / 16;
  constexpr int STAGE = (BM + BN) * 128;             // bytes of one K-step of 32
  constexpr int AP = BM * 8 / T, BP = BN * 8 / T;    // 16-byte loads a thread and K-step
  constexpr int SLD = WN + 2;
  static_assert(AP * T == BM * 8 && BP * T == BN * 8 && MI % 2 == 0, "tile and threads");
  static_assert(T / 64 * 32 * SLD * 4 <= NST * STAGE, "the slabs fit the stages' LDS");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WGN, wn = wave % WGN;
  const NsWork w = ns_work<BM, BN, EPI>(mats, tb, ws, p, xcd_remap(blockIdx.x, gridDim.x));

  // a wave loads halves of blocks, a kilobyte each.  Blocks past the matrix are read from its last rows: their products
  // are not stored.
  const int nk = w.K / 32;
  const char* ga[AP];
  const char* gb[BP];
#pragma unroll
  for (int i = 0; i < AP; ++i) {
    const int q = i * (T / 64) + wave;
    ga[i] = w.A + (long)min(w.m0 / 16 + (q >> 1), w.dest.rows / 16 - 1) * nk * 2048 + (q & 1) * 1024 + lane * 16;
  }
#pragma unroll
  for (int i = 0; i < BP; ++i) {
    const int q = i * (T / 64) + wave;
    gb[i] = w.B + (long)min(w.n0 / 16 + (q >> 1), w.dest.cols / 16 - 1) * nk * 2048 + (q & 1) * 1024 + lane * 16;
  }
  auto stage = [&](int kt, int buf) {
    char* l = smem + buf * STAGE + wave * 1024;
#pragma unroll
    for (int i = 0; i < AP; ++i) glds16(ga[i] + (long)kt * 2048, l + i * T * 16);
#pragma unroll
    for (int i = 0; i < BP; ++i) glds16(gb[i] + (long)kt * 2048, l + BM * 128 + i * T * 16);
  };
  const int fhi = lane * 16, flo = 1024 + lane * 16;

  f32x4_t acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

  const char* sa = smem + wm * WM * 128;
  const char* sb = smem + (BM + wn * WN) * 128;
#define NS_MMA_ROW(i, AH, AL, bh, bl)                                                                                          \
  _Pragma("unroll") for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bl[j], AH, acc[i][j], 0, 0, 0); \
  _Pragma("unroll") for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], AL, acc[i][j], 0, 0, 0); \
  _Pragma("unroll") for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], AH, acc[i][j], 0, 0, 0);
  f16x8_t ah[2][MI], al[2][MI], bh[2][NI], bl[2][NI];
#define NS_READ(u, at)                                                                              \
  {                                                                                                 \
  const char *a_ = sa + (at) * STAGE, *b_ = sb + (at) * STAGE;                                    \
  _Pragma("unroll") for (int j = 0; j < NI; ++j) {                                                \
    bh[u][j] = *(const f16x8_t*)(b_ + j * 2048 + fhi);                                            \
    bl[u][j] = *(const f16x8_t*)(b_ + j * 2048 + flo);                                            \
  }                                                                                               \
  _Pragma("unroll") for (int i = 0; i < MI; ++i) {                                                \
    ah[u][i] = *(const f16x8_t*)(a_ + i * 2048 + fhi);                                            \
    al[u][i] = *(const f16x8_t*)(a_ + i * 2048 + flo);                                            \
  }                                                                                               \
  }
#pragma unroll
  for (int k = 0; k < NST; ++k)
    if (k < nk) stage(k, k);
  // stage 0 has landed when at most the others are under way
  if (NST <= nk) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * (AP + BP)) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  NS_READ(0, 0)
  int buf = 0;
  for (int kt = 0; kt < nk; kt += 2) {             // K is a multiple of 64
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // this step's fragments are here, and stage kt + u + 1 has landed: at most NST - 2 younger ones are under way
      if (kt + u + NST - 1 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * (AP + BP)) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();                // everybody has read stage kt + u: its place is free
      asm volatile("" ::: "memory");
      if (kt + u + NST < nk) stage(kt + u + NST, buf);
      buf = buf + 1 == NST ? 0 : buf + 1;
      NS_READ(u ^ 1, buf)                          // (behind the last step: old values, not used)
#pragma unroll
      for (int i = 0; i < MI; ++i) { NS_MMA_ROW(i, ah[u][i], al[u][i], bh[u], bl[u]) }
      // a read between every three matrix instructions: in one go they hold up the wave's issue
#pragma unroll
      for (int i = 0; i < 2 * (MI + NI); ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, MI * NI * 3 / (2 * (MI + NI)), 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    }
  }
#undef NS_READ
#undef NS_MMA_ROW
  __syncthreads();                                   // every wave is done with the stages: the slabs go there

  ns_store<MI, NI, EPI>(mats[w.mat], p, w.dest, acc, w.m0 + wm * WM, w.n0 + wn * WN, (uint32_t*)smem + wave * 32 * SLD);
}

// Small tiles, where a launch has few of them and the time from the first load to the last store counts: a workgroup's
// four waves share out K, not the tile.  A wave multiplies all of the 16F x 16F tile for every fourth K-step, with its
// fragments loaded straight into registers, S - 1 steps ahead: no LDS, no barrier in the loop, 3F matrix instructions for
// four loads.  The waves' sums meet in LDS.  Where tiles are far fewer than CUs and K is long, K is cut between
// workgroups too (nsplit): they leave their sums in `slabs` and ns_finish_kernel adds them up.  (Adding them up in the
// last workgroup to arrive needs a device-wide fence from each: 62 us instead of 28 for the Gram matrix of 512 x 4608.)
template <int F, int EPI>
__global__ __launch_bounds__(256, 1) void ns_tile_kernel(const NsMat* __restrict__ mats, const NsBlocks tb, char* __restrict__ ws, const NsGemm p) {
  constexpr int S = F == 4 ? 3 : 6;
  __shared__ __attribute__((aligned(16))) f32x4_t part[4][F * F][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // shared tiles: K's eighths go to the eight XCDs (blocks go round them), so that each L2 sees an eighth of the operands
  const int block = tb.shared ? (int)blockIdx.x : xcd_remap(blockIdx.x, gridDim.x);
  const NsWork w = ns_work<16 * F, 16 * F, EPI>(mats, tb, ws, p, block);
  const int nk = w.K / 32, first = wave + 4 * w.split, stride = 4 * w.nsplit;
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(w.A + (long)w.m0 * nk * 128, F * 16L * nk * 128);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(w.B + (long)w.n0 * nk * 128, F * 16L * nk * 128);
  const int steps = first < nk ? (nk - first + stride - 1) / stride : 0;
  const unsigned hi = lane * 16, lo = 1024 + lane * 16;

  f32x4_t acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  f16x8_t ah[S][F], al[S][F], bh[S][F], bl[S][F];
#define NS_LOAD(u, step)                                                                                             \
  {                                                                                                                  \
    _Pragma("unroll") for (int i = 0; i < F; ++i) {                                                                  \
      const int at_ = (i * nk + first + (step) * stride) * 2048;                                                     \
      bl[u][i] = __builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(rb, lo, at_, 0));                 \
      ah[u][i] = __builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(ra, hi, at_, 0));                 \
      bh[u][i] = __builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(rb, hi, at_, 0));                 \
      al[u][i] = __builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(ra, lo, at_, 0));                 \
    }                                                                                                                \
  }
#define NS_MMA(u)                                                                                                    \
  {                                                                                                                  \
    _Pragma("unroll") for (int i = 0; i < F; ++i) _Pragma("unroll") for (int j = 0; j < F; ++j) acc[i][j] =          \
        __builtin_amdgcn_mfma_f32_16x16x32_f16(bl[u][j], ah[u][i], acc[i][j], 0, 0, 0);                              \
    _Pragma("unroll") for (int i = 0; i < F; ++i) _Pragma("unroll") for (int j = 0; j < F; ++j) acc[i][j] =          \
        __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[u][j], al[u][i], acc[i][j], 0, 0, 0);                              \
    _Pragma("unroll") for (int i = 0; i < F; ++i) _Pragma("unroll") for (int j = 0; j < F; ++j) acc[i][j] =          \
        __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[u][j], ah[u][i], acc[i][j], 0, 0, 0);                              \
  }
  // Set u's products with the loads of set v between them, one behind every 3F/4 matrix instructions: issued in one go
  // they hold up the wave, and its SIMD has no other.
#define NS_STEP(u, v, step)                                                                                          \
  {                                                                                                                  \
    _Pragma("unroll") for (int q = 0; q < 3 * F * F; ++q) {                                                          \
      const int i = q % (F * F) / F, j = q % F;                                                                      \
      if (q < F * F) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bl[u][j], ah[u][i], acc[i][j], 0, 0, 0);     \
      else if (q < 2 * F * F) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[u][j], al[u][i], acc[i][j], 0, 0, 0); \
      else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[u][j], ah[u][i], acc[i][j], 0, 0, 0);               \
      if (q * 4 % (3 * F) < 4) {                                                                                     \
        const int l = q * 4 / (3 * F), x = l % F, at_ = (x * nk + first + (step) * stride) * 2048;                   \
        if (l < F) bl[v][x] = __builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(rb, lo, at_, 0));    \
        else if (l < 2 * F) ah[v][x] = __builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(ra, hi, at_, 0)); \
        else if (l < 3 * F) bh[v][x] = __builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(rb, hi, at_, 0)); \
        else al[v][x] = __builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(ra, lo, at_, 0));          \
        __builtin_amdgcn_sched_barrier(0);                                                                           \
      }                                                                                                              \
    }                                                                                                                \
  }
  // no condition on a load in the loop: behind one, hipcc no longer counts what is under way and waits for all of it
  if (steps >= S) {
#pragma unroll
    for (int u = 0; u < S - 1; ++u) NS_LOAD(u, u)
    int k = 0;
    for (; k + 2 * S - 1 <= steps; k += S) {
#pragma unroll
      for (int u = 0; u < S; ++u) NS_STEP(u, (u + S - 1) % S, k + u + S - 1)
    }
#pragma unroll
    for (int u = 0; u < 2 * S - 2; ++u) {
      if (k + u + S - 1 < steps) NS_LOAD((u + S - 1) % S, k + u + S - 1)
      if (k + u < steps) NS_MMA(u % S)
    }
  } else {
#pragma unroll
    for (int u = 0; u < S - 1; ++u)
      if (u < steps) NS_LOAD(u, u)
#pragma unroll
    for (int u = 0; u < S - 1; ++u)
      if (u < steps) NS_MMA(u)
  }
#undef NS_STEP
#undef NS_MMA
#undef NS_LOAD
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j) part[wave][i * F + j][lane] = acc[i][j];
  __syncthreads();
  // a wave goes on with 32 x 32 of the tile: a quadrant, or (F = 2) the first wave with all of it
  if (wave >= F * F / 4) return;
  const int wi = wave >> 1, wj = wave & 1;
  f32x4_t sum[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int f = (wi * 2 + i) * F + wj * 2 + j;
      sum[i][j] = (part[0][f][lane] + part[1][f][lane]) + (part[2][f][lane] + part[3][f][lane]);
    }
  if (w.nsplit > 1) {
    f32x4_t* slab = (f32x4_t*)(ws + NS_AT_SLABS) + ((size_t)block * (F * F / 4) + wave) * 256 + lane;
#pragma unroll
    for (int f = 0; f < 4; ++f) slab[f * 64] = sum[f >> 1][f & 1];
    return;
  }
  __shared__ uint32_t slabs[F * F / 4][32 * 34];
  ns_store<2, 2, EPI>(mats[w.mat], p, w.dest, sum, w.m0 + wi * 32, w.n0 + wj * 32, slabs[wave]);
}

// Adds up the shared tiles' sums in order: a wave for 32 x 32
template <int F>
__global__ __launch_bounds__(64) void ns_finish_kernel(const NsMat* __restrict__ mats, const NsBlocks tb, char* __restrict__ ws, const NsGemm p) {
  __shared__ uint32_t mine[32 * 34];
  constexpr int Q = F * F / 4;
  const int lane = threadIdx.x, q = blockIdx.x % Q, block = blockIdx.x / Q * NS_SPLIT;
  const NsWork w = ns_work<16 * F, 16 * F, EPI_PAIR>(mats, tb, ws, p, block);
  const f32x4_t* slab = (const f32x4_t*)(ws + NS_AT_SLABS) + ((size_t)block * Q + q) * 256 + lane;
  f32x4_t sum[2][2];
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    f32x4_t v = slab[f * 64];
#pragma unroll
    for (int k = 1; k < NS_SPLIT; ++k) v += slab[(size_t)k * Q * 256 + f * 64];
    sum[f >> 1][f & 1] = v;
  }
  ns_store<2, 2, EPI_PAIR>(mats[w.mat], p, w.dest, sum, w.m0 + (q >> 1) * 32, w.n0 + (q & 1) * 32, mine);
}

// The whole of it in one workgroup a matrix, for m <= 128: twenty launches of 4 us each, most of it start and end, are
// what a small matrix costs in the kernels above.  A and P live in LDS (two buffers of at most 64 KB, in the layout
// above), Q as fragments in the registers of the waves that own its rows; R, the next A and the next Q wait in
// accumulators until their place is free.  X is read from G where it is needed and turned into pairs on the way; between
// segments it is in the workspace, f32 [m][n].  Eight waves as 4 x 2.
struct NsSmall {
  float scale[44];                                   // of every segment: X, then A, P, Q of its steps
  float coef[3], eps;
  int steps, out_kind;
};

// Steps of each segment: at most three, as even as they go, longer ones first.
__host__ __device__ inline int segment_steps(int steps, int seg) {
  const int n = (steps + 2) / 3;
  return steps / n + (seg < steps % n ? 1 : 0);
}

// scale / |G| as mantissa and power of two: the number itself leaves f32 for |G| below 2.4e-35 (a zero matrix times
// infinity), and v * 2^e first is exact.
struct NsFactor { float mant; int e; };

// 8 values of X along memory or across it: elements i0, i0 + stride, ... of G, `have` of them (the rest zero)
template <int KIND, int MUON>
DTP_DEVINL void ns_load8(const NsMat& t, const MuonArgs& ma, const long i0, const int stride, const int have,
                         const NsFactor inv, float* v) {
  float m[8];
  if (stride == 1 && have == 8 && t.aligned && (i0 & 7) == 0) {
    if (KIND == 0) {
      const f32x4_t a = *(const f32x4_t*)((const float*)t.src + i0), b = *(const f32x4_t*)((const float*)t.src + i0 + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
    } else if (KIND == 1) {
      const u32x4_t a = *(const u32x4_t*)((const bf16_t*)t.src + i0);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(a[e] << 16); v[2 * e + 1] = __uint_as_float(a[e] & 0xFFFF0000u); }
    } else {
      const f16x8_t a = *(const f16x8_t*)((const f16_t*)t.src + i0);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
    }
    if (MUON) {
      const f32x4_t a = *(const f32x4_t*)(t.mom + i0), b = *(const f32x4_t*)(t.mom + i0 + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { m[e] = a[e]; m[4 + e] = b[e]; }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = e < have;
      v[e] = in ? load_as_f32<KIND>(t.src, i0 + (long)e * stride) : 0.f;
      if (MUON) m[e] = in ? t.mom[i0 + (long)e * stride] : 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (MUON) v[e] = muon_again(v[e], m[e], ma);
    v[e] = ldexpf(v[e], inv.e) * inv.mant;
  }
}

DTP_DEVINL void ns_pairs(const float* v, f16x8_t& hi, f16x8_t& lo) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f16_t h, l;
    split_f16(v[e], h, l);
    hi[e] = h;
    lo[e] = l;
  }
}

template <int MP, int KIND, int MUON>
__global__ __launch_bounds__(512) void ns_small_kernel(const NsTable tb, char* __restrict__ ws, const NsSmall q, const MuonArgs ma) {
  constexpr int MI = MP / 64, NI = MP / 32, KS = MP / 32, RB = MP / 16;     // a wave's tile, K-steps, 16-row blocks
  constexpr int SUP = 32 / RB;                                              // K-steps of X staged at a time: 64 KB
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  __shared__ double red[8];
  char *B1 = smem, *B2 = smem + 65536;
  const NsMat& t = tb.mat[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, frow = lane & 15, fk = lane >> 4;
  const bool tall = t.rows > t.cols;
  const int mr = tall ? t.cols : t.rows, nr = tall ? t.rows : t.cols;       // real sides
  float* X1 = (float*)(ws + t.off[0]);

  // ---- the norm (muon: momentum on the way)
  double sq = 0.0;
  const long total = (long)t.rows * t.cols;
#pragma unroll 4
  for (long i = tid; i < total; i += 512) {
    float u = load_as_f32<KIND>(t.src, i);
    if (MUON) {
      float m = t.mom[i];
      u = muon_direction(u, m, ma);
      t.mom[i] = m;
    }
    sq += (double)u * (double)u;
  }
  sq = wave_sum_f64(sq);
  if (lane == 0) red[wave] = sq;
  __syncthreads();
  sq = 0.0;
  for (int i = 0; i < 8; ++i) sq += red[i];
  const double norm = sqrt(sq) + (double)q.eps;

  f32x4_t acc[MI][NI], accq[MI][NI];
  f16x8_t qh[MI][KS], ql[MI][KS];
#define NS_FRAG(buf, rb, ks, half) (*(const f16x8_t*)((buf) + ((rb) * KS + (ks)) * 2048 + (half) * 1024 + lane * 16))
#define NS_ZERO(c) \
  _Pragma("unroll") for (int i = 0; i < MI; ++i) _Pragma("unroll") for (int j = 0; j < NI; ++j) c[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#define NS_MMA3(c, AH, AL, bh, bl) \
  _Pragma("unroll") for (int i = 0; i < MI; ++i) _Pragma("unroll") for (int j = 0; j < NI; ++j) c[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bl[j], AH, c[i][j], 0, 0, 0); \
  _Pragma("unroll") for (int i = 0; i < MI; ++i) _Pragma("unroll") for (int j = 0; j < NI; ++j) c[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], AL, c[i][j], 0, 0, 0); \
  _Pragma("unroll") for (int i = 0; i < MI; ++i) _Pragma("unroll") for (int j = 0; j < NI; ++j) c[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], AH, c[i][j], 0, 0, 0);
  auto product = [&](const char* A, const char* B) {               // acc = this wave's tile of A B
    NS_ZERO(acc)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      f16x8_t ah[MI], al[MI], bh[NI], bl[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j) { bh[j] = NS_FRAG(B, wn * NI + j, ks, 0); bl[j] = NS_FRAG(B, wn * NI + j, ks, 1); }
#pragma unroll
      for (int i = 0; i < MI; ++i) { ah[i] = NS_FRAG(A, wm * MI + i, ks, 0); al[i] = NS_FRAG(A, wm * MI + i, ks, 1); }
      NS_MMA3(acc, ah[i], al[i], bh, bl)
      if (MP > 64) asm volatile("" ::: "memory");        // one K-step's fragments at a time: registers
    }
  };
  // where a lane's four values of fragment (i, j) lie in a buffer
  auto place = [&](int i, int j) { return ((wm * MI + i) * KS + ((wn * NI + j) >> 1)) * 2048 + (frow + 16 * (((wn * NI + j) & 1) * 2 + (fk >> 1))) * 16 + (fk & 1) * 8; };
  auto put = [&](f32x4_t (&c)[MI][NI], char* to, float scale) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const f32x4_t v = c[i][j] * scale;
        const f16x4_t hi = __builtin_convertvector(v, f16x4_t);
        const f16x4_t lo = __builtin_convertvector(v - __builtin_convertvector(hi, f32x4_t), f16x4_t);
        char* d = to + place(i, j);
        *(f16x4_t*)d = hi;
        *(f16x4_t*)(d + 1024) = lo;
      }
  };

  int sc = 0;                                        // this segment's scales
  const int nseg = (q.steps + 2) / 3;
  for (int seg = 0; seg < nseg; ++seg) {
    const int ns = segment_steps(q.steps, seg);
    const float sx = q.scale[sc];
    NsFactor inv0;
    inv0.mant = (float)frexp((double)sx / norm, &inv0.e);
    // 8 neighbouring values along n of row r of X, times its scale
    auto load_x = [&](int r, int k, float* v) {
      if (seg == 0) {
        const int have = r < mr ? min(8, nr - k) : 0;
        ns_load8<KIND, MUON>(t, ma, tall ? (long)k * t.cols + r : (long)r * t.cols + k, tall ? t.cols : 1, have, inv0, v);
      } else {
        const f32x4_t a = *(const f32x4_t*)(X1 + (long)r * t.n + k), b = *(const f32x4_t*)(X1 + (long)r * t.n + k + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = a[e] * sx; v[4 + e] = b[e] * sx; }
      }
    };
    // ---- A = X X^T
    float sa = q.scale[sc + 1];
    NS_ZERO(acc)
    const int nk = t.n / 32;
    for (int k0 = 0; k0 < nk; k0 += SUP) {
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int b = wave * 4 + f, rb = b / SUP, ks = b % SUP;
        if (k0 + ks < nk) {
          float v[8];
          load_x(rb * 16 + frow, (k0 + ks) * 32 + fk * 8, v);
          f16x8_t hi, lo;
          ns_pairs(v, hi, lo);
          *(f16x8_t*)(smem + b * 2048 + lane * 16) = hi;
          *(f16x8_t*)(smem + b * 2048 + 1024 + lane * 16) = lo;
        }
      }
      __syncthreads();
      const int have = min(SUP, nk - k0);
      for (int ks = 0; ks < have; ++ks) {
#define NS_STAGED(rb, half) (*(const f16x8_t*)(smem + ((rb) * SUP + ks) * 2048 + (half) * 1024 + lane * 16))
        f16x8_t ah[MI], al[MI], bh[NI], bl[NI];
#pragma unroll
        for (int j = 0; j < NI; ++j) { bh[j] = NS_STAGED(wn * NI + j, 0); bl[j] = NS_STAGED(wn * NI + j, 1); }
#pragma unroll
        for (int i = 0; i < MI; ++i) { ah[i] = NS_STAGED(wm * MI + i, 0); al[i] = NS_STAGED(wm * MI + i, 1); }
        NS_MMA3(acc, ah[i], al[i], bh, bl)
#undef NS_STAGED
      }
      __syncthreads();
    }
    put(acc, B1, sa / (sx * sx));
    __syncthreads();
    // ---- the polynomials
    float sqs = 0.f;
    for (int k = 0; k < ns; ++k) {
      const bool last = k + 1 == ns;
      const float sqn = q.scale[sc + 3 * k + 3], sp = k == 0 ? sqn : q.scale[sc + 3 * k + 2];       // the first step's P is its Q
      product(B1, B1);
      const float s2 = q.coef[2] * sp / (sa * sa), s1 = q.coef[1] * sp / sa, s0 = q.coef[0] * sp;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const char* a = B1 + place(i, j);
          const f32x4_t av = __builtin_convertvector(*(const f16x4_t*)a, f32x4_t) + __builtin_convertvector(*(const f16x4_t*)(a + 1024), f32x4_t);
          acc[i][j] = acc[i][j] * s2 + av * s1;
          const int r = (wm * MI + i) * 16 + frow, c = (wn * NI + j) * 16 + fk * 4;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e == r) acc[i][j][e] += s0;
        }
      put(acc, B2, 1.f);
      __syncthreads();
      if (k > 0) {                                   // Q P, from the old Q's rows
        NS_ZERO(accq)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          f16x8_t bh[NI], bl[NI];
#pragma unroll
          for (int j = 0; j < NI; ++j) { bh[j] = NS_FRAG(B2, wn * NI + j, ks, 0); bl[j] = NS_FRAG(B2, wn * NI + j, ks, 1); }
          NS_MMA3(accq, qh[i][ks], ql[i][ks], bh, bl)
          if (MP > 64) asm volatile("" ::: "memory");
        }
      }
      if (!last) {
        const float san = q.scale[sc + 3 * k + 4];
        product(B2, B1);                             // R = P A, at A's scale
        __syncthreads();
        put(acc, B1, 1.f / sp);
        __syncthreads();
        product(B2, B1);                             // A = P R
        __syncthreads();
        put(acc, B1, san / (sp * sa));
        sa = san;
      } else {
        __syncthreads();
      }
      if (k > 0) put(accq, B2, sqn / (sp * sqs));
      __syncthreads();
      if (!last) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) { qh[i][ks] = NS_FRAG(B2, wm * MI + i, ks, 0); ql[i][ks] = NS_FRAG(B2, wm * MI + i, ks, 1); }
        __syncthreads();
      }
      sqs = sqn;
    }
    // ---- Q X: a wave takes 16 columns of X at a time
    const bool final_ = seg + 1 == nseg, turned = final_ && tall;
    const float so = 1.f / (sqs * sx);
    for (int nb = wave; nb < t.n / 16; nb += 8) {
      f16x8_t xh[KS], xl[KS];
      const int c = nb * 16 + frow;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float v[8];
        const int k = ks * 32 + fk * 8;              // 8 neighbouring values along m of column c
        if (seg == 0) {
          const int have = c < nr ? max(0, min(8, mr - k)) : 0;
          ns_load8<KIND, MUON>(t, ma, tall ? (long)c * t.cols + k : (long)k * t.cols + c, tall ? 1 : t.cols, have, inv0, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = X1[(long)(k + e) * t.n + c] * sx;
        }
        ns_pairs(v, xh[ks], xl[ks]);
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll 1
      for (int rb = 0; rb < RB; ++rb) {
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const f16x8_t h = NS_FRAG(B2, rb, ks, 0), l = NS_FRAG(B2, rb, ks, 1);
          if (turned) {                              // rows of O are X's columns
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(l, xh[ks], o, 0, 0, 0);
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, xl[ks], o, 0, 0, 0);
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(h, xh[ks], o, 0, 0, 0);
          } else {
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl[ks], h, o, 0, 0, 0);
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh[ks], l, o, 0, 0, 0);
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh[ks], h, o, 0, 0, 0);
          }
        }
        o = o * so;
        const int r = turned ? nb * 16 + frow : rb * 16 + frow, cc = turned ? rb * 16 + fk * 4 : nb * 16 + fk * 4;
        if (final_) {
          ns_out(t, q.out_kind, r, cc, o);
        } else {
          *(f32x4_t*)(X1 + (long)r * t.n + cc) = o;
        }
      }
    }
    sc += 1 + 3 * ns;
    __syncthreads();
  }
#undef NS_FRAG
#undef NS_ZERO
#undef NS_MMA3
}

int round64(int v) { return (v + 63) / 64 * 64; }
long align256(long v) { return (v + 255) / 256 * 256; }

struct NsCall {
  NsTable tb;
  int count;
  char* ws;
  hipStream_t st;
};

// fills the padded sides and offsets; returns the workspace's bytes
long ns_layout(NsCall& c) {
  long at = NS_AT_MATS;
  for (int i = 0; i < c.count; ++i) {
    NsMat& t = c.tb.mat[i];
    const int a = round64(t.rows), b = round64(t.cols);
    const bool tall = t.rows > t.cols;
    t.m = tall ? b : a;
    t.n = tall ? a : b;
    t.off[0] = at;
    at = align256(at + 3L * t.m * t.n * 4);
    t.off[1] = at;
    at = align256(at + 5L * t.m * t.m * 4);
  }
  return at;
}

template <int EPI> long tiles(const NsCall& c, const NsGemm& p, int i, int bm, int bn) {
  const NsMat& t = c.tb.mat[i];
  const bool swap = EPI == EPI_OUT && t.rows > t.cols;
  const long rows = swap ? t.n : t.m, cols = p.is_long && !swap ? t.n : t.m;
  const long tr = (rows + bm - 1) / bm, tc = (cols + bn - 1) / bn;
  return p.nops * (p.is_long || EPI == EPI_OUT ? tr * tc : tr * (tr + 1) / 2);
}

template <int BM, int BN, int WGM, int WGN, int NST, int EPI>
int launch_gemm(const NsCall& c, const NsGemm& p) {
  NsBlocks bl = {};
  long at = 0;
  for (int i = 0; i < c.count; ++i) {
    bl.first[i] = (int)at;
    at += tiles<EPI>(c, p, i, BM, BN);
  }
  if (at > 0x7fffffffL) return -14;
  bl.first[bl.count = c.count] = (int)at;
  const int lds = NST * (BM + BN) * 128;
  const auto k = ns_gemm_kernel<BM, BN, WGM, WGN, NST, EPI>;
  if (lds > 65536 && hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return -2;
  hipLaunchKernelGGL(k, dim3((unsigned)at), dim3(WGM * WGN * 64), lds, c.st, (const NsMat*)c.ws, bl, c.ws, p);
  return DTP_CHECK_LAUNCH();
}

template <int F, int EPI> int launch_tiles(const NsCall& c, const NsGemm& p, bool shared) {
  NsBlocks bl = {};
  long at = 0;
  for (int i = 0; i < c.count; ++i) {
    bl.first[i] = (int)at;
    at += tiles<EPI>(c, p, i, 16 * F, 16 * F) * (shared ? NS_SPLIT : 1);
  }
  if (at > 0x7fffffffL || (shared && at > NS_SHARED * NS_SPLIT)) return -14;
  bl.first[bl.count = c.count] = (int)at;
  bl.shared = shared;
  hipLaunchKernelGGL((ns_tile_kernel<F, EPI>), dim3((unsigned)at), dim3(256), 0, c.st, (const NsMat*)c.ws, bl, c.ws, p);
  if (shared)
    hipLaunchKernelGGL((ns_finish_kernel<F>), dim3((unsigned)(at / NS_SPLIT * (F * F / 4))), dim3(64), 0, c.st, (const NsMat*)c.ws,
                       bl, c.ws, p);
  return DTP_CHECK_LAUNCH();
}

// Tile by the time it takes to work through the launch: rounds of 256 workgroups (one a CU) times the tile's cost.  Costs
// in units of a 64 x 64 tile's, from chains of equal products: 2048 x 2048 (us in all) 128: 888, 64: 889, 32: 994, 192:
// 1315; 4096 x 4096 192: 3659, 64: 4878, 128: 4996, 32: 7166; 1024 x 1024 64: 220, 32: 263, 128: 487; 512 x 512 32: 6.2
// a product, 64: 8.3.
// shared: whether K is cut between workgroups.
template <int EPI> int tile_side(const NsCall& c, const NsGemm& p, bool& shared) {
  const int side[4] = {192, 128, 64, 32};
  const double cost[4] = {5.5, 3.0, 1.0, 0.4};
  long n[4];
  int best = 3;
  for (int v = 3; v >= 0; --v) {
    n[v] = 0;
    for (int i = 0; i < c.count; ++i) n[v] += tiles<EPI>(c, p, i, side[v], side[v]);
    if ((double)((n[v] + 255) / 256) * cost[v] < (double)((n[best] + 255) / 256) * cost[best]) best = v;
  }
  shared = false;
  if (EPI == EPI_PAIR && p.op[0].a == W_X && n[2] <= NS_SHARED) {
    // few tiles and a long K (the Gram matrix of 512 x 4608): 17 us shared out, adding up included; 28 otherwise
    int nk = 0;
    for (int i = 0; i < c.count; ++i) nk = nk < c.tb.mat[i].n / 32 ? c.tb.mat[i].n / 32 : nk;
    shared = nk >= 64;
  }
  return shared ? 64 : side[best];
}

template <int EPI> int gemm(const NsCall& c, const NsGemm& p) {
  bool shared;
  const int side = tile_side<EPI>(c, p, shared);
  if (side == 192) return launch_gemm<192, 192, 2, 4, 3, EPI>(c, p);
  if (side == 128) return launch_gemm<128, 128, 2, 2, 4, EPI>(c, p);
  if (side == 32) return launch_tiles<2, EPI>(c, p, false);
  if (EPI == EPI_PAIR && shared) return launch_tiles<4, EPI_PAIR>(c, p, true);
  return launch_tiles<4, EPI>(c, p, false);
}

template <int KIND, int MUON>
int ns_front(const NsCall& c, const MuonArgs& ma, float eps, float scale) {
  NsBlocks bl = {};
  long at = 0;
  for (int i = 0; i < c.count; ++i) {
    bl.first[i] = (int)at;
    at += norm_blocks(c.tb.mat[i].rows, c.tb.mat[i].cols);
  }
  bl.first[bl.count = c.count] = (int)at;
  hipLaunchKernelGGL((ns_norm_kernel<KIND, MUON>), dim3((unsigned)at), dim3(256), 0, c.st, c.tb, bl, c.ws, ma);
  at = 0;
  for (int i = 0; i < c.count; ++i) {
    bl.first[i] = (int)at;
    at += (long)(c.tb.mat[i].m / 64) * (c.tb.mat[i].n / 64);
  }
  if (at > 0x7fffffffL) return -14;
  bl.first[c.count] = (int)at;
  hipLaunchKernelGGL((ns_split_kernel<KIND, MUON>), dim3((unsigned)at), dim3(256), 0, c.st, (const NsMat*)c.ws, bl, c.ws,
                     (const double*)(c.ws + NS_AT_PART), ma, eps, scale);
  return DTP_CHECK_LAUNCH();
}

int ns_chain(const NsCall& c, int steps, const float* coeffs, const float* scales, int out_kind);

// One workgroup a matrix: where every m is at most 128 and no long side keeps a single CU busy for longer than the
// launches it saves.
// 64 x 576 takes 50 us here and 86 in launches, 64 x 1152 89 and 89; 128 x 128 60 and 89, 128 x 576 128 and 92.
// (All matrices of a part have to be small enough: one that is not takes the others along into the launches, and the
// last bits of a result depend on the way.)
bool ns_is_small(const NsCall& c) {
  for (int i = 0; i < c.count; ++i)
    if (c.tb.mat[i].m > 128 || c.tb.mat[i].n > (c.tb.mat[i].m > 64 ? 320 : 1088)) return false;
  return true;
}

template <int KIND, int MUON>
int ns_small(const NsCall& c, const MuonArgs& ma, int steps, const float* coeffs, const float* scales, float eps, int out_kind) {
  NsSmall q = {};
  const int n = (steps + 2) / 3 + 3 * steps;
  if (n > (int)(sizeof(q.scale) / sizeof(float))) return -12;
  for (int i = 0; i < n; ++i) q.scale[i] = scales[i];
  for (int i = 0; i < 3; ++i) q.coef[i] = coeffs[i];
  q.eps = eps;
  q.steps = steps;
  q.out_kind = out_kind;
  bool wide = false;
  for (int i = 0; i < c.count; ++i) wide |= c.tb.mat[i].m > 64;
  const int lds = 131072;
  const auto k = wide ? ns_small_kernel<128, KIND, MUON> : ns_small_kernel<64, KIND, MUON>;
  if (hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return -2;
  hipLaunchKernelGGL(k, dim3(c.count), dim3(512), lds, c.st, c.tb, c.ws, q, ma);
  return DTP_CHECK_LAUNCH();
}

template <int KIND, int MUON>
int ns_run(const NsCall& c, const MuonArgs& ma, int steps, const float* coeffs, const float* scales, float eps, int out_kind) {
  if (ns_is_small(c)) return ns_small<KIND, MUON>(c, ma, steps, coeffs, scales, eps, out_kind);
  const int rc = ns_front<KIND, MUON>(c, ma, eps, scales[0]);
  return rc ? rc : ns_chain(c, steps, coeffs, scales, out_kind);
}

// coeffs: a, b, c.  scales: powers of two that the matrices are held at: for every segment X, then for each of its
// steps A, P, Q.
int ns_chain(const NsCall& c, int steps, const float* coeffs, const float* scales, int out_kind) {
  const int nseg = (steps + 2) / 3;
  NsGemm p = {};
  int rc, xt = W_XT0;
  for (int seg = 0; seg < nseg; ++seg) {
    const int ns = segment_steps(steps, seg);
    const float sx = scales[0];
    float sa = scales[1], sq = 0.f;
    p.nops = 1;
    p.is_long = 0;
    p.op[0] = {W_X, W_X, W_A, -1, sa / (sx * sx)};
    if ((rc = gemm<EPI_PAIR>(c, p))) return rc;
    int q = W_Q0;
    for (int k = 0; k < ns; ++k) {
      const bool last = k + 1 == ns;
      const float sqn = scales[3 * k + 3];
      const int P = k == 0 ? q : W_P;                  // the first step's P is its Q
      const float sp = k == 0 ? sqn : scales[3 * k + 2];
      p.nops = 1;
      p.op[0] = {W_A, W_A, P, -1, coeffs[2] * sp / (sa * sa)};
      p.ca = coeffs[0] * sp;
      p.cb = coeffs[1] * sp / sa;
      if ((rc = gemm<EPI_POLY>(c, p))) return rc;
      const int qn = q == W_Q0 ? W_Q1 : W_Q0;
      p.nops = 0;
      if (!last) p.op[p.nops++] = {P, W_A, W_R, -1, 1.f / sp};                   // R at A's scale
      if (k > 0) p.op[p.nops++] = {P, q, qn, -1, sqn / (sp * sq)};
      if (p.nops && (rc = gemm<EPI_PAIR>(c, p))) return rc;
      if (!last) {
        const float san = scales[3 * k + 4];
        p.nops = 1;
        p.op[0] = {P, W_R, W_A, -1, san / (sp * sa)};
        if ((rc = gemm<EPI_PAIR>(c, p))) return rc;
        sa = san;
      }
      if (k > 0) q = qn;
      sq = sqn;
    }
    scales += 1 + 3 * ns;
    p.nops = 1;
    p.is_long = 1;
    if (seg + 1 < nseg) {
      const int to = xt == W_XT0 ? W_XT1 : W_XT0;      // X^T is read here: its successor goes next to it
      p.op[0] = {q, xt, W_X, to, scales[0] / (sq * sx)};
      if ((rc = gemm<EPI_PAIR>(c, p))) return rc;
      xt = to;
    } else {
      p.out_kind = out_kind;
      p.op[0] = {q, xt, 0, -1, 1.f / (sq * sx)};
      if ((rc = gemm<EPI_OUT>(c, p))) return rc;
    }
  }
  return 0;
}

int fill_table(NsCall& c, int count, const int* rows, const int* cols) {
  if (count < 1 || count > NS_MAXMAT) return -10;
  c.count = count;
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 1 || cols[i] < 1 || rows[i] > (1 << 20) || cols[i] > (1 << 20)) return -11;
    c.tb.mat[i] = NsMat{};
    c.tb.mat[i].rows = rows[i];
    c.tb.mat[i].cols = cols[i];
  }
  return 0;
}

// A matrix with m above 1024 is worked off alone, the others of a call together; the parts follow one another on the stream
// and share the workspace.  Measured in a list (us; VGG16's thirteen convolution weights and one more, alone / in every
// launch with them): 1100 x 1100 603 / 664, 1408 x 1408 643 / 806, 2048 x 2048 1179 / 1390,
// 4096 x 4096 3913 / 5486 (XCDs whose tiles have a shorter K wait for the others).  Where all matrices of a call are alike
// nothing waits, and the rule costs time: two of 1024 x 1024 414 / 363, three of 1100 x 1100 711 / 528, two of 2048 x 2048
// 1624 / 1386, of 4096 x 4096 7030 / 7218.
constexpr int NS_ALONE = 1024;

template <class F> int each_part(const NsCall& all, F run) {
  NsCall part = all;
  int rc = 0, k = 0;
  for (int i = 0; i < all.count; ++i) {
    const NsMat& t = all.tb.mat[i];
    if ((t.rows < t.cols ? t.rows : t.cols) > NS_ALONE) {
      NsCall one = all;
      one.count = 1;
      one.tb.mat[0] = t;
      if ((rc = run(one))) return rc;
    } else {
      part.tb.mat[k++] = t;
    }
  }
  part.count = k;
  return k ? run(part) : 0;
}

long ns_bytes(const NsCall& all) {
  long most = 0;
  each_part(all, [&](NsCall& c) {
    const long n = ns_layout(c);
    if (n > most) most = n;
    return 0;
  });
  return most;
}

}  // namespace

// Bytes of scratch for these matrices (at most 24 a call); 0: refused.
extern "C" size_t dtp_ns_workspace(int count, const int* rows, const int* cols) {
  NsCall c;
  if (fill_table(c, count, rows, cols)) return 0;
  return (size_t)ns_bytes(c);
}

// Tile side that a product of one matrix's chain is worked off in (by launches; matrices for one workgroup have none: 0).
// product: 0 the Gram matrix, 1 the polynomial, 2 P A and P Q together, 3 Q X between segments, 4 the last Q X.
extern "C" int dtp_ns_tile(int rows, int cols, int product) {
  NsCall c;
  if (fill_table(c, 1, &rows, &cols) || product < 0 || product > 4) return -10;
  ns_layout(c);
  if (ns_is_small(c)) return 0;
  NsGemm p = {};
  bool shared;
  p.nops = product == 2 ? 2 : 1;
  p.is_long = product >= 3;
  p.op[0].a = product == 0 ? W_X : W_P;
  return product == 1 ? tile_side<EPI_POLY>(c, p, shared) : product == 4 ? tile_side<EPI_OUT>(c, p, shared)
                                                                          : tile_side<EPI_PAIR>(c, p, shared);
}

// out[i] = Newton-Schulz of src[i] ([rows][cols], contiguous).  in_kind / out_kind: 0 f32, 1 bf16, 2 f16.
// scales: powers of two, see ns_chain.  ws: dtp_ns_workspace bytes, 256-byte aligned.
extern "C" int dtp_newton_schulz(int count, const void** src, void** out, const int* rows, const int* cols, int in_kind,
                                 int out_kind, int steps, const float* coeffs, const float* scales, float eps, void* ws,
                                 size_t ws_bytes, hipStream_t st) {
  NsCall all;
  const int rc = fill_table(all, count, rows, cols);
  if (rc) return rc;
  if (steps < 1 || in_kind < 0 || in_kind > 2 || out_kind < 0 || out_kind > 2) return -12;
  if ((size_t)ns_bytes(all) > ws_bytes) return -13;
  for (int i = 0; i < count; ++i) {
    NsMat& t = all.tb.mat[i];
    t.src = src[i];
    t.out = out[i];
    t.aligned = (((size_t)src[i] | (size_t)out[i]) & 15) == 0;
  }
  const MuonArgs ma = {};
  all.ws = (char*)ws;
  all.st = st;
  return each_part(all, [&](NsCall& c) {
    ns_layout(c);
    return in_kind == 0 ? ns_run<0, 0>(c, ma, steps, coeffs, scales, eps, out_kind)
           : in_kind == 1 ? ns_run<1, 0>(c, ma, steps, coeffs, scales, eps, out_kind)
                          : ns_run<2, 0>(c, ma, steps, coeffs, scales, eps, out_kind);
  });
}

// One Muon step: mom <- momentum*mom + (1-momentum)*grad; O = Newton-Schulz of (nesterov ? (1-momentum)*grad +
// momentum*mom : mom); w <- w*decay[i] - step[i]*O; lp[i] = bf16(w) where given.  grad_bf16: gradient type.
extern "C" int dtp_muon_step(int count, void** w, const void** grad, void** mom, void** lp, const int* rows,
                             const int* cols, int grad_bf16, float momentum, int nesterov, float grad_scale,
                             const float* decay, const float* step, int steps, const float* coeffs, const float* scales,
                             float eps, void* ws, size_t ws_bytes, hipStream_t st) {
  NsCall all;
  const int rc = fill_table(all, count, rows, cols);
  if (rc) return rc;
  if (steps < 1) return -12;
  if ((size_t)ns_bytes(all) > ws_bytes) return -13;
  for (int i = 0; i < count; ++i) {
    NsMat& t = all.tb.mat[i];
    t.src = grad[i]; t.mom = (float*)mom[i]; t.w = (float*)w[i]; t.out = lp[i];
    t.decay = decay[i]; t.step = step[i];
    t.aligned = (((size_t)grad[i] | (size_t)mom[i] | (size_t)w[i] | (size_t)lp[i]) & 15) == 0;
  }
  const MuonArgs ma = {momentum, 1.f - momentum, grad_scale, nesterov};
  all.ws = (char*)ws;
  all.st = st;
  return each_part(all, [&](NsCall& c) {
    ns_layout(c);
    return grad_bf16 ? ns_run<1, 1>(c, ma, steps, coeffs, scales, eps, 3) : ns_run<0, 1>(c, ma, steps, coeffs, scales, eps, 3);
  });
}
