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
// segment of five, a^5 = 484, is 1e-3 off for a matrix of rank one where a loop of f32 products is 5e-5 off, and
// 3 + 2 is 5e-5 off too.  And every matrix is held as a pair of f16 values, hi + lo (22 bits), scaled by a power of
// two into f16's range; a product of two of them is three MFMA products, hi*hi + hi*lo + lo*hi, accumulated in f32
// (lo*lo is 2^-22 of the sum).  Single 16-bit values would be 1e-2 and more off.
//
// Pair layout of a [rows][K] matrix: K in blocks of 32; a block of a row is 32 hi values, then their 32 lo values:
// 128 bytes, one cache line, one row of an LDS tile.
#include "dtp_common.h"

namespace {

typedef _Float16 f16_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;

constexpr int NS_MAXMAT = 24;            // matrices per call: their table travels as a kernel argument
constexpr int NS_PART = 1024;            // partial sums of squares per matrix

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
};

struct NsTable {
  NsMat mat[NS_MAXMAT];
  int first[NS_MAXMAT + 1];      // first block of each matrix in this launch
  int count;
};

DTP_DEVINL char* ws_at(char* ws, const NsMat& t, int which) {
  if (which <= W_XT1) return ws + t.off[0] + (long)which * t.m * t.n * 4;
  return ws + t.off[1] + (long)(which - W_A) * t.m * t.m * 4;
}

DTP_DEVINL int find_mat(const NsTable& tb, int block) {
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

// element (r, k) of a pair matrix of ld columns: offset of its hi value, in f16; lo is 32 further
DTP_DEVINL long pair_at(long r, int k, int ld) { return r * 2 * ld + (k >> 5) * 64 + (k & 31); }

template <int KIND> DTP_DEVINL float load_as_f32(const void* p, long i) {   // 0 f32, 1 bf16, 2 f16
  if (KIND == 0) return ((const float*)p)[i];
  if (KIND == 1) return bf16_to_f32(((const bf16_t*)p)[i]);
  return (float)((const f16_t*)p)[i];
}

struct MuonArgs { float mu, omu, gscale; int nesterov; };      // omu = 1 - momentum

DTP_DEVINL double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Sum of squares of G in f64 (any magnitude of G: no overflow, nothing lost on 10^8 values), one partial a block.
// Muon: momentum <- mu*momentum + (1-mu)*grad on the way; G = nesterov ? (1-mu)*grad + mu*momentum : momentum.
template <int KIND, int MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsTable tb, double* __restrict__ part, const MuonArgs ma) {
  __shared__ double red[4];
  const int mi = find_mat(tb, blockIdx.x);
  const NsMat& t = tb.mat[mi];
  const int b = blockIdx.x - tb.first[mi], nb = tb.first[mi + 1] - tb.first[mi];
  const long total = (long)t.rows * t.cols;
  double s = 0.0;
  for (long i = (long)b * 256 + threadIdx.x; i < total; i += (long)nb * 256) {
    float u = load_as_f32<KIND>(t.src, i);
    if (MUON) {
      u *= ma.gscale;
      const float mo = fmaf(ma.omu, u, ma.mu * t.mom[i]);
      t.mom[i] = mo;
      u = ma.nesterov ? fmaf(ma.mu, mo, ma.omu * u) : mo;
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
__global__ __launch_bounds__(256) void ns_split_kernel(const NsTable tb, char* __restrict__ ws,
                                                       const double* __restrict__ part, const MuonArgs ma,
                                                       const float eps, const float scale) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int mi = find_mat(tb, blockIdx.x);
  const NsMat& t = tb.mat[mi];
  const bool tall = t.rows > t.cols;
  const int pr = tall ? t.n : t.m, pc = tall ? t.m : t.n;          // padded rows / columns of G
  const int b = blockIdx.x - tb.first[mi], tc = pc / 64, br = b / tc, bc = b - br * tc;
  const int nparts = norm_blocks(t.rows, t.cols);
  double s = 0.0;
  for (int i = threadIdx.x; i < nparts; i += 256) s += part[mi * NS_PART + i];
  s = wave_sum_f64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const double inv = (double)scale / (sqrt(red[0] + red[1] + red[2] + red[3]) + (double)eps);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  f16_t* same = (f16_t*)ws_at(ws, t, tall ? W_XT0 : W_X);
  f16_t* turn = (f16_t*)ws_at(ws, t, tall ? W_X : W_XT0);
  for (int r = wave; r < 64; r += 4) {
    const int gr = br * 64 + r, gc = bc * 64 + lane;
    float u = 0.f;
    if (gr < t.rows && gc < t.cols) {
      const long i = (long)gr * t.cols + gc;
      u = load_as_f32<KIND>(t.src, i);
      if (MUON) {
        u *= ma.gscale;
        const float mo = t.mom[i];
        u = ma.nesterov ? fmaf(ma.mu, mo, ma.omu * u) : mo;
      }
      u = (float)((double)u * inv);
    }
    tile[r][lane] = u;
    f16_t hi, lo;
    split_f16(u, hi, lo);
    const long o = pair_at(gr, gc, pc);
    same[o] = hi;
    same[o + 32] = lo;
  }
  __syncthreads();
  for (int c = wave; c < 64; c += 4) {
    f16_t hi, lo;
    split_f16(tile[lane][c], hi, lo);
    const long o = pair_at(bc * 64 + c, br * 64 + lane, pr);
    turn[o] = hi;
    turn[o + 32] = lo;
  }
}

// One product of pair matrices per matrix of the table: D = A B^T, both operands [rows][K] in pair layout.
struct NsOp { int a, b, d, dt; float scale; };       // operands, result, its transpose (-1: none), factor from the accumulator
struct NsGemm {
  NsOp op[2];
  int nops;
  int out_kind;                                      // EPI_OUT: 0 f32, 1 bf16, 2 f16, 3 muon
  float ca, cb;                                      // EPI_POLY: result = ca I + cb * A + scale * acc
};

enum { EPI_PAIR = 0, EPI_POLY = 1, EPI_OUT = 2 };

template <int BM, int BN, int WGM, int WGN, int EPI>
__global__ __launch_bounds__(WGM * WGN * 64) void ns_gemm_kernel(const NsTable tb, char* __restrict__ ws, const NsGemm p) {
  constexpr int T = WGM * WGN * 64;
  constexpr int WM = BM / WGM, WN = BN / WGN, MI = WM / 16, NI = WN / 16;
  constexpr int STAGE = (BM + BN) * 128;             // bytes of one K-step of 32
  constexpr int AP = BM * 8 / T, BP = BN * 8 / T;    // 16-byte loads a thread and K-step
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WGN, wn = wave % WGN;
  const int mi = find_mat(tb, blockIdx.x);
  const NsMat& t = tb.mat[mi];
  const bool tall = t.rows > t.cols;
  int b = blockIdx.x - tb.first[mi];
  const int per = (tb.first[mi + 1] - tb.first[mi]) / p.nops, oi = b / per;
  b -= oi * per;
  const NsOp op = p.op[oi];
  // EPI_OUT: O = Q X_0 for a wide G, O = X_0^T Q for a tall one: rows and columns of O are G's
  const bool swap = EPI == EPI_OUT && tall;
  const int asel = swap ? op.b : op.a, bsel = swap ? op.a : op.b;
  const int rows = swap ? t.n : t.m, cols = swap || op.b > W_XT1 || op.b == W_X ? t.m : t.n;
  const int K = asel == W_X ? t.n : t.m;             // the Gram product runs along the long side
  const int tn = (cols + BN - 1) / BN;
  const int m0 = (b / tn) * BM, n0 = (b % tn) * BN;

  // LDS image: 128-byte rows (one pair block), 16-byte chunk c of row r at c ^ ((r >> 1) & 7).  Rows past the
  // matrix are read from its last row: their products are not stored.
  const char* ga[AP];
  const char* gb[BP];
  const char* A = ws_at(ws, t, asel);
  const char* B = ws_at(ws, t, bsel);
#pragma unroll
  for (int i = 0; i < AP; ++i) {
    const int idx = i * T + tid, r = idx >> 3, c = (idx & 7) ^ ((r >> 1) & 7);
    ga[i] = A + (long)min(m0 + r, rows - 1) * K * 4 + c * 16;
  }
#pragma unroll
  for (int i = 0; i < BP; ++i) {
    const int idx = i * T + tid, r = idx >> 3, c = (idx & 7) ^ ((r >> 1) & 7);
    gb[i] = B + (long)min(n0 + r, cols - 1) * K * 4 + c * 16;
  }
  auto stage = [&](int kt, int buf) {
    char* l = smem + buf * STAGE + wave * 1024;
#pragma unroll
    for (int i = 0; i < AP; ++i) glds16(ga[i] + (long)kt * 128, l + i * T * 16);
#pragma unroll
    for (int i = 0; i < BP; ++i) glds16(gb[i] + (long)kt * 128, l + BM * 128 + i * T * 16);
  };
  const int frow = lane & 15, fk = lane >> 4, fsw = (frow >> 1) & 7;
  const int fhi = frow * 128 + ((fk ^ fsw) << 4), flo = frow * 128 + (((4 + fk) ^ fsw) << 4);

  f32x4_t acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

  const int nk = K / 32;
  stage(0, 0);
  for (int kt = 0; kt < nk; ++kt) {
    sync_lds_dma();
    if (kt + 1 < nk) stage(kt + 1, (kt + 1) & 1);
    const char* sa = smem + (kt & 1) * STAGE + wm * WM * 128;
    const char* sb = smem + (kt & 1) * STAGE + (BM + wn * WN) * 128;
    f16x8_t bh[NI], bl[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      bh[j] = *(const f16x8_t*)(sb + j * 2048 + fhi);
      bl[j] = *(const f16x8_t*)(sb + j * 2048 + flo);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const f16x8_t ah = *(const f16x8_t*)(sa + i * 2048 + fhi);
      const f16x8_t al = *(const f16x8_t*)(sa + i * 2048 + flo);
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bl[j], ah, acc[i][j], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], al, acc[i][j], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], ah, acc[i][j], 0, 0, 0);
    }
  }

  // a lane holds row m0 + wm*WM + i*16 + (lane & 15), columns n0 + wn*WN + j*16 + (lane >> 4) * 4 + 0..3
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int r = m0 + wm * WM + i * 16 + frow;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int c = n0 + wn * WN + j * 16 + fk * 4;
      f32x4_t v = acc[i][j] * op.scale;
      if (EPI == EPI_OUT) {
        if (r >= t.rows) continue;
        const long o = (long)r * t.cols + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (c + e >= t.cols) continue;
          if (p.out_kind == 0) ((float*)t.out)[o + e] = v[e];
          else if (p.out_kind == 1) ((bf16_t*)t.out)[o + e] = f32_to_bf16(v[e]);
          else if (p.out_kind == 2) ((f16_t*)t.out)[o + e] = (f16_t)v[e];
          else {
            const float w = fmaf(t.w[o + e], t.decay, -t.step * v[e]);
            t.w[o + e] = w;
            if (t.out) ((bf16_t*)t.out)[o + e] = f32_to_bf16(w);
          }
        }
      } else {
        if (r >= rows || c >= cols) continue;
        const long o = pair_at(r, c, cols);
        if (EPI == EPI_POLY) {
          const f16_t* q = (const f16_t*)A + o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = fmaf(p.cb, (float)q[e] + (float)q[e + 32], v[e]);
            if (c + e == r) v[e] += p.ca;
          }
        }
        f16_t* d = (f16_t*)ws_at(ws, t, op.d) + o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f16_t hi, lo;
          split_f16(v[e], hi, lo);
          d[e] = hi;
          d[e + 32] = lo;
          if (op.dt >= 0) {
            f16_t* dt = (f16_t*)ws_at(ws, t, op.dt) + pair_at(c + e, r, rows);
            dt[0] = hi;
            dt[32] = lo;
          }
        }
      }
    }
  }
}

int round64(int v) { return (v + 63) / 64 * 64; }
long align256(long v) { return (v + 255) / 256 * 256; }

// fills the padded sides and offsets; returns the workspace's bytes
long ns_layout(NsTable& tb) {
  long at = (long)tb.count * NS_PART * 8;
  for (int i = 0; i < tb.count; ++i) {
    NsMat& t = tb.mat[i];
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

long tiles(const NsTable& tb, const NsGemm& p, int i, int bm, int bn, bool out) {
  const NsMat& t = tb.mat[i];
  const bool is_long = p.op[0].b == W_XT0 || p.op[0].b == W_XT1, swap = out && t.rows > t.cols;
  const long rows = swap ? t.n : t.m, cols = is_long && !swap ? t.n : t.m;
  return p.nops * ((rows + bm - 1) / bm) * ((cols + bn - 1) / bn);
}

template <int BM, int BN, int WGM, int WGN, int EPI>
int launch_gemm(NsTable& tb, char* ws, const NsGemm& p, hipStream_t st) {
  long at = 0;
  for (int i = 0; i < tb.count; ++i) {
    tb.first[i] = (int)at;
    at += tiles(tb, p, i, BM, BN, EPI == EPI_OUT);
  }
  if (at > 0x7fffffffL) return -14;
  tb.first[tb.count] = (int)at;
  const int lds = 2 * (BM + BN) * 128;
  const auto k = ns_gemm_kernel<BM, BN, WGM, WGN, EPI>;
  if (lds > 65536 && hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return -2;
  hipLaunchKernelGGL(k, dim3((unsigned)at), dim3(WGM * WGN * 64), lds, st, tb, ws, p);
  return DTP_CHECK_LAUNCH();
}

// The largest tile that still gives about half the CUs one.
template <int EPI> int gemm(NsTable& tb, char* ws, const NsGemm& p, hipStream_t st) {
  long t256 = 0, t128 = 0;
  for (int i = 0; i < tb.count; ++i) {
    t256 += tiles(tb, p, i, 256, 256, EPI == EPI_OUT);
    t128 += tiles(tb, p, i, 128, 128, EPI == EPI_OUT);
  }
  if (t256 >= 128) return launch_gemm<256, 256, 2, 4, EPI>(tb, ws, p, st);
  if (t128 >= 128) return launch_gemm<128, 128, 2, 2, EPI>(tb, ws, p, st);
  return launch_gemm<64, 64, 2, 2, EPI>(tb, ws, p, st);
}

template <int KIND, int MUON>
int ns_front(NsTable& tb, char* ws, const MuonArgs& ma, float eps, float scale, hipStream_t st) {
  double* part = (double*)ws;
  long at = 0;
  for (int i = 0; i < tb.count; ++i) {
    tb.first[i] = (int)at;
    at += norm_blocks(tb.mat[i].rows, tb.mat[i].cols);
  }
  tb.first[tb.count] = (int)at;
  hipLaunchKernelGGL((ns_norm_kernel<KIND, MUON>), dim3((unsigned)at), dim3(256), 0, st, tb, part, ma);
  at = 0;
  for (int i = 0; i < tb.count; ++i) {
    tb.first[i] = (int)at;
    at += (long)(tb.mat[i].m / 64) * (tb.mat[i].n / 64);
  }
  if (at > 0x7fffffffL) return -14;
  tb.first[tb.count] = (int)at;
  hipLaunchKernelGGL((ns_split_kernel<KIND, MUON>), dim3((unsigned)at), dim3(256), 0, st, tb, ws, part, ma, eps, scale);
  return DTP_CHECK_LAUNCH();
}

// Steps of each segment: at most three, as even as they go, longer ones first.
int segment_steps(int steps, int seg) {
  const int n = (steps + 2) / 3;
  return steps / n + (seg < steps % n ? 1 : 0);
}

// coeffs: a, b, c.  scales: powers of two that the matrices are held at: for every segment X, then for each of its
// steps A, P, Q.
int ns_chain(NsTable& tb, char* ws, int steps, const float* coeffs, const float* scales, int out_kind, hipStream_t st) {
  const int nseg = (steps + 2) / 3;
  NsGemm p = {};
  int rc, xt = W_XT0;
  for (int seg = 0; seg < nseg; ++seg) {
    const int ns = segment_steps(steps, seg);
    const float sx = scales[0];
    float sa = scales[1], sq = 0.f;
    p.nops = 1;
    p.op[0] = {W_X, W_X, W_A, -1, sa / (sx * sx)};
    if ((rc = gemm<EPI_PAIR>(tb, ws, p, st))) return rc;
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
      if ((rc = gemm<EPI_POLY>(tb, ws, p, st))) return rc;
      const int qn = q == W_Q0 ? W_Q1 : W_Q0;
      p.nops = 0;
      if (!last) p.op[p.nops++] = {P, W_A, W_R, -1, 1.f / sp};                   // R at A's scale
      if (k > 0) p.op[p.nops++] = {P, q, qn, -1, sqn / (sp * sq)};
      if (p.nops && (rc = gemm<EPI_PAIR>(tb, ws, p, st))) return rc;
      if (!last) {
        const float san = scales[3 * k + 4];
        p.nops = 1;
        p.op[0] = {P, W_R, W_A, -1, san / (sp * sa)};
        if ((rc = gemm<EPI_PAIR>(tb, ws, p, st))) return rc;
        sa = san;
      }
      if (k > 0) q = qn;
      sq = sqn;
    }
    scales += 1 + 3 * ns;
    p.nops = 1;
    if (seg + 1 < nseg) {
      const int to = xt == W_XT0 ? W_XT1 : W_XT0;      // X^T is read here: its successor goes next to it
      p.op[0] = {q, xt, W_X, to, scales[0] / (sq * sx)};
      if ((rc = gemm<EPI_PAIR>(tb, ws, p, st))) return rc;
      xt = to;
    } else {
      p.out_kind = out_kind;
      p.op[0] = {q, xt, 0, -1, 1.f / (sq * sx)};
      if ((rc = gemm<EPI_OUT>(tb, ws, p, st))) return rc;
    }
  }
  return 0;
}

int fill_table(NsTable& tb, int count, const int* rows, const int* cols) {
  if (count < 1 || count > NS_MAXMAT) return -10;
  tb.count = count;
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 1 || cols[i] < 1 || rows[i] > (1 << 20) || cols[i] > (1 << 20)) return -11;
    tb.mat[i] = NsMat{};
    tb.mat[i].rows = rows[i];
    tb.mat[i].cols = cols[i];
  }
  return 0;
}

}  // namespace

// Bytes of scratch for these matrices (at most 24 a call); 0: refused.
extern "C" size_t dtp_ns_workspace(int count, const int* rows, const int* cols) {
  NsTable tb;
  if (fill_table(tb, count, rows, cols)) return 0;
  return (size_t)ns_layout(tb);
}

// out[i] = Newton-Schulz of src[i] ([rows][cols], contiguous).  in_kind / out_kind: 0 f32, 1 bf16, 2 f16.
// scales: powers of two, see ns_chain.  ws: dtp_ns_workspace bytes, 256-byte aligned.
extern "C" int dtp_newton_schulz(int count, const void** src, void** out, const int* rows, const int* cols, int in_kind,
                                 int out_kind, int steps, const float* coeffs, const float* scales, float eps, void* ws,
                                 size_t ws_bytes, hipStream_t st) {
  NsTable tb;
  int rc = fill_table(tb, count, rows, cols);
  if (rc) return rc;
  if (steps < 1 || in_kind < 0 || in_kind > 2 || out_kind < 0 || out_kind > 2) return -12;
  if ((size_t)ns_layout(tb) > ws_bytes) return -13;
  for (int i = 0; i < count; ++i) { tb.mat[i].src = src[i]; tb.mat[i].out = out[i]; }
  const MuonArgs ma = {};
  char* w = (char*)ws;
  rc = in_kind == 0 ? ns_front<0, 0>(tb, w, ma, eps, scales[0], st)
       : in_kind == 1 ? ns_front<1, 0>(tb, w, ma, eps, scales[0], st) : ns_front<2, 0>(tb, w, ma, eps, scales[0], st);
  if (rc) return rc;
  return ns_chain(tb, w, steps, coeffs, scales, out_kind, st);
}

// One Muon step: mom <- momentum*mom + (1-momentum)*grad; O = Newton-Schulz of (nesterov ? (1-momentum)*grad +
// momentum*mom : mom); w <- w*decay[i] - step[i]*O; lp[i] = bf16(w) where given.  grad_bf16: gradient type.
extern "C" int dtp_muon_step(int count, void** w, const void** grad, void** mom, void** lp, const int* rows,
                             const int* cols, int grad_bf16, float momentum, int nesterov, float grad_scale,
                             const float* decay, const float* step, int steps, const float* coeffs, const float* scales,
                             float eps, void* ws, size_t ws_bytes, hipStream_t st) {
  NsTable tb;
  int rc = fill_table(tb, count, rows, cols);
  if (rc) return rc;
  if (steps < 1) return -12;
  if ((size_t)ns_layout(tb) > ws_bytes) return -13;
  for (int i = 0; i < count; ++i) {
    NsMat& t = tb.mat[i];
    t.src = grad[i]; t.mom = (float*)mom[i]; t.w = (float*)w[i]; t.out = lp[i];
    t.decay = decay[i]; t.step = step[i];
  }
  const MuonArgs ma = {momentum, 1.f - momentum, grad_scale, nesterov};
  char* wsb = (char*)ws;
  rc = grad_bf16 ? ns_front<1, 1>(tb, wsb, ma, eps, scales[0], st) : ns_front<0, 1>(tb, wsb, ma, eps, scales[0], st);
  if (rc) return rc;
  return ns_chain(tb, wsb, steps, coeffs, scales, 3, st);
}
