// Orthogonalisation of small matrices and of matrices with one short side.
//
// Both sides at most 128 (k_orth_direct): x and A stay in LDS in fp32, a workgroup per matrix does all steps as they are defined on
// v_mfma_f32_16x16x4, one launch. Bound by the chain of products, reads from LDS and barriers of a step (40 x 40: 21 tiles of 10 matrix
// instructions, 2 us; 190 matrices, eight steps: 21 us).
//
// A short side m of at most 64, the other longer: all steps of x <- (a + b A + c A A) x, A = x x', act on x from the short side, so
//   x_T = Q x_0,   P = a I + b A + c A A,   Q <- P Q,   A <- P A P
// needs the m x n matrix twice (for A_0 = x_0 x_0' and for the last product) whatever the number of steps; |g|_F^2 is the trace of g g'.
// In exact arithmetic that is the definition. In floating point an error of A_0 grows with the square of a small singular value's growth
// (five steps of a = 3.4445: a^8 = 2e4 relative to the largest), which fp32 cannot pay and fp64 can: the m x m side and both products run
// on v_mfma_f64_16x16x4 (below 64 rows they cost less than reading x does; the entries of x convert exactly). Not for any number of steps:
// a singular value of zero leaves an eigenvalue of about -1e-17, and one that has grown to -0.1 runs off to infinity (nothing pulls a negative one
// back; a newly formed A = x x' has none). orth_run bounds that growth from the coefficients; where it ends (after eleven of the steps above) the
// product is written in fp32 and the next run starts from it.
// A, P, Q commute and are symmetric: tiles on and below the diagonal are computed and mirrored, those of A in themselves too. Left as it comes
// out of the product of A P and P, A's upper half would differ from the lower one by roundings there, and that difference grows by a^3 a step
// (in eight steps of the above to 6e-6 of a low-rank matrix, in twelve to 20; mirrored 4e-11 and 8e-9).
//   n up to 1024, or many matrices: everything in one workgroup per matrix, one launch (k_orth_small).
//   longer: partial sums of g g' over slices (k_orth_gram, k_orth_gram_sum), the steps in one workgroup (k_orth_steps), the product
//   (k_orth_apply). 100 000 x 40 in fp32, eight steps: 14 + 4 + 35 + 22 us. The steps are a chain of fp64 products on one CU (4 us each),
//   the passes over x are bound by HBM (1.1 and 1.4 TB/s: fp64 matrix instructions and 16 MB, too little to fill it).
#include <algorithm>
#include <cmath>

#include "dense_dev.h"

namespace scl {

typedef double f64x4 __attribute__((ext_vector_type(4)));

struct SmallArgs {
  OrthArgs o;  // coef: device pointer is not needed, the steps' coefficients ride in `coef`
  int tall, m, slices;
  int start;  // x is the caller's and is divided by its norm first
  int64_t n;
  double* part;  // [batch][slices][tiles * 256]
  double* gram;  // [batch][tiles * 256]
  double* Q;     // [batch][16 MT][16 MT]
};
constexpr int MAX_RIDE = 24;  // steps whose coefficients fit the kernel's arguments
struct Coefs { double v[3 * MAX_RIDE]; };

template <int MT> struct Tiles {
  static constexpr int R = 16 * MT, LQ = R + 2, LI = R + 1, NL = MT * (MT + 1) / 2;
  // doubles of LDS for A, P, Q, which hold the waves' partial sums of A first
  static constexpr int WORK = 3 * R * LQ > 4 * NL * 256 ? 3 * R * LQ : 4 * NL * 256;
};
// the t-th tile on or below the diagonal, by rows
__device__ __forceinline__ void lower_tile(int t, int* i, int* j) {
  int r = 0;
  while ((r + 1) * (r + 2) / 2 <= t) ++r;
  *i = r;
  *j = t - r * (r + 1) / 2;
}

// Where a thread's 4 MT elements of 16 NW columns of x lie: below the columns' first element in x and y (in 32 bits: orth_is_small), and
// in Xs[k][i]. Computed once: the divisions by R cost more than the loads.
template <int MT, int NW>
struct Places {
  unsigned in[4 * MT], out[4 * MT];
  unsigned short at[4 * MT], k[4 * MT];  // k: column, 0xffff for rows behind m
  __device__ __forceinline__ Places(const SmallArgs& a) {
    constexpr int R = 16 * MT, CK = 16 * NW, LI = R + 1;
#pragma unroll
    for (int e = 0; e < 4 * MT; ++e) {
      const int id = e * (64 * NW) + (int)threadIdx.x;
      const int i = a.tall ? id % R : id / CK, c = a.tall ? id / R : id % CK;
      at[e] = (unsigned short)(c * LI + i);
      k[e] = (unsigned short)(i < a.m ? c : 0xffff);
      in[e] = (unsigned)(a.tall ? c * a.o.ldx + i : i * a.o.ldx + c);
      out[e] = (unsigned)(a.tall ? c * a.o.ldy + i : i * a.o.ldy + c);
    }
  }
};
// columns k0 .. of x (zeros outside) into registers, then into Xs
template <int T, int MT, int NW>
struct Slab {
  float v[4 * MT];
  __device__ __forceinline__ void fetch(const SmallArgs& a, const Places<MT, NW>& pl, int64_t b, int64_t k0, int64_t kend) {
    const auto* p = static_cast<const typename Elem<T>::type*>(a.o.x) + b * a.o.sx + (a.tall ? k0 * a.o.ldx : k0);
    const int n = (int)min((int64_t)(16 * NW), kend - k0);
#pragma unroll
    for (int e = 0; e < 4 * MT; ++e) v[e] = pl.k[e] < n ? Elem<T>::ld(p + pl.in[e]) : 0.f;
  }
  __device__ __forceinline__ void put(const Places<MT, NW>& pl, float* Xs) {
#pragma unroll
    for (int e = 0; e < 4 * MT; ++e) Xs[pl.at[e]] = v[e];
  }
};

// red[tile][g * 64 + lane] = sum over k0 <= k < kend of x x' (unscaled); every wave takes 16 of the columns in Xs. Loads run up to three
// slabs ahead. part: 4 * NL * 256 doubles of LDS (the waves' sums, waves 4 .. 7 added to 0 .. 3 first, then those in order).
template <int T, int MT, int NW>
__device__ __forceinline__ void gram_range(const SmallArgs& a, int64_t b, int64_t k0, int64_t kend, float* Xs, double* part, double* red) {
  constexpr int LI = Tiles<MT>::LI, NL = Tiles<MT>::NL, CK = 16 * NW;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
  f64x4 acc[NL];
#pragma unroll
  for (int t = 0; t < NL; ++t) acc[t] = f64x4{0, 0, 0, 0};
  const Places<MT, NW> pl(a);
  constexpr int PF = MT == 4 && NW == 8 ? 1 : 3;  // (more would not fit the registers)
  Slab<T, MT, NW> s[PF];
#pragma unroll
  for (int u = 0; u < PF; ++u)
    if (k0 + u * CK < kend) s[u].fetch(a, pl, b, k0 + u * CK, kend);
  for (int64_t k = k0; k < kend; k += PF * CK) {
#pragma unroll
    for (int u = 0; u < PF; ++u) {
      const int64_t ku = k + u * CK;
      if (ku < kend) {
        s[u].put(pl, Xs);
        __syncthreads();
        if (ku + PF * CK < kend) s[u].fetch(a, pl, b, ku + PF * CK, kend);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          double f[MT];
#pragma unroll
          for (int i = 0; i < MT; ++i) f[i] = (double)Xs[(wid * 16 + ks * 4 + q) * LI + i * 16 + r16];
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) acc[i * (i + 1) / 2 + j] = __builtin_amdgcn_mfma_f64_16x16x4f64(f[i], f[j], acc[i * (i + 1) / 2 + j], 0, 0, 0);
        }
        __syncthreads();
      }
    }
  }
  auto slot = [&](int t, int g) -> double& { return part[((wid & 3) * NL + t) * 256 + g * 64 + lane]; };
#pragma unroll
  for (int r = NW / 4 - 1; r >= 0; --r) {
    if (wid / 4 == r) {
#pragma unroll
      for (int t = 0; t < NL; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) slot(t, g) = r == NW / 4 - 1 ? acc[t][g] : acc[t][g] + slot(t, g);
    }
    __syncthreads();
  }
  for (int e = threadIdx.x; e < NL * 256; e += 64 * NW)
    red[e] = (part[e] + part[NL * 256 + e]) + (part[2 * NL * 256 + e] + part[3 * NL * 256 + e]);
  __syncthreads();
}

// C tile (i, j) = X Y for symmetric X, Y in LDS: all reads first, then the chain of matrix instructions (64 cycles each) up to column m
template <int MT>
__device__ __forceinline__ f64x4 tile_product(const double* X, const double* Y, int i, int j, int m) {
  constexpr int LQ = Tiles<MT>::LQ, KS = 4 * MT;
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const double *x = X + (i * 16 + r16) * LQ + q, *y = Y + (j * 16 + r16) * LQ + q;
  double xv[KS], yv[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    xv[s] = x[4 * s];
    yv[s] = y[4 * s];
  }
  __builtin_amdgcn_sched_barrier(0);
  f64x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};  // (two chains: one alone waits for itself)
#pragma unroll
  for (int s = 0; s < KS; ++s)
    if (s < 4 * (MT - 1) || 4 * s < m) acc[s & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64(xv[s], yv[s], acc[s & 1], 0, 0, 0);
  return acc[0] + acc[1];
}
template <int MT, bool EXACT = false>  // EXACT: a tile on the diagonal is made symmetric
__device__ __forceinline__ void tile_store(double* C, int i, int j, f64x4 v) {
  constexpr int LQ = Tiles<MT>::LQ;
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int r = i * 16 + q + 4 * g, c = j * 16 + r16;
    if (!EXACT || r >= c) C[r * LQ + c] = v[g];
    if (EXACT ? r > c : i != j) C[c * LQ + r] = v[g];
  }
}

// from the sums in `red` to Q (with the 1 / (|g|_F + eps) of x_0 in it); 8 waves
template <int MT>
__device__ __forceinline__ void steps(const SmallArgs& a, const Coefs& cf, const double* red, double* A, double* P, double* Q, double* scal) {
  constexpr int R = Tiles<MT>::R, LQ = Tiles<MT>::LQ, NL = Tiles<MT>::NL, NT = (NL + 7) / 8;
  const int tid = threadIdx.x, wid = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r16 = lane & 15, q = lane >> 4;
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const int t = wid + 8 * u;
    if (t < NL) {
      int i, j;
      lower_tile(t, &i, &j);
      f64x4 v;
#pragma unroll
      for (int g = 0; g < 4; ++g) v[g] = red[t * 256 + g * 64 + lane];
      tile_store<MT>(A, i, j, v);
    }
  }
  __syncthreads();
  if (tid == 0) {
    double s = 0.0;
    for (int i = 0; i < a.m; ++i) s += A[i * LQ + i];
    scal[0] = a.start ? 1.0 / (sqrt(s) + a.o.eps) : 1.0;
  }
  __syncthreads();
  const double f = scal[0];
  for (int e = tid; e < R * R; e += 512) {
    const int r = e / R, c = e % R;
    A[r * LQ + c] *= f * f;
    Q[r * LQ + c] = r == c && r < a.m ? f : 0.0;
  }
  __syncthreads();
  // (tiles are dealt out to the 8 waves, two of which share a SIMD: the 12 of the second phase at m = 40 are 3 per SIMD)
  for (int t = 0; t < a.o.steps; ++t) {
    const double ca = cf.v[3 * t], cb = cf.v[3 * t + 1], cc = cf.v[3 * t + 2];
    const bool last = t + 1 == a.o.steps;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int w = wid + 8 * u;
      if (w < NL) {
        int i, j;
        lower_tile(w, &i, &j);
        f64x4 v = tile_product<MT>(A, A, i, j, a.m);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int r = i * 16 + q + 4 * g, c = j * 16 + r16;
          v[g] = cc * v[g] + cb * A[r * LQ + c] + (r == c && r < a.m ? ca : 0.0);
        }
        tile_store<MT>(P, i, j, v);
      }
    }
    __syncthreads();
    // P Q and, but for the last step, A P
    constexpr int N2 = (2 * NL + 7) / 8;
    f64x4 v2[N2];
#pragma unroll
    for (int u = 0; u < N2; ++u) {
      const int w = wid + 8 * u;
      if (w < (last ? NL : 2 * NL)) {
        int i, j;
        lower_tile(w < NL ? w : w - NL, &i, &j);
        v2[u] = tile_product<MT>(w < NL ? Q : A, P, i, j, a.m);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < N2; ++u) {
      const int w = wid + 8 * u;
      if (w < (last ? NL : 2 * NL)) {
        int i, j;
        lower_tile(w < NL ? w : w - NL, &i, &j);
        tile_store<MT>(w < NL ? Q : A, i, j, v2[u]);
      }
    }
    __syncthreads();
    if (last) break;
    f64x4 va[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int w = wid + 8 * u;
      if (w < NL) {
        int i, j;
        lower_tile(w, &i, &j);
        va[u] = tile_product<MT>(A, P, i, j, a.m);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int w = wid + 8 * u;
      if (w < NL) {
        int i, j;
        lower_tile(w, &i, &j);
        tile_store<MT, true>(A, i, j, va[u]);
      }
    }
    __syncthreads();
  }
}

// y = Q x for k0 <= k < kend, 16 NW columns at a time; Q [R][ldq] in LDS. y may be x: columns are read before they are written.
template <int T, int U, int MT, int NW>
__device__ __forceinline__ void apply_range(const SmallArgs& a, int64_t b, int64_t k0, int64_t kend, float* Xs, const double* Q) {
  constexpr int R = Tiles<MT>::R, LQ = Tiles<MT>::LQ, LI = Tiles<MT>::LI, CK = 16 * NW;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
  constexpr int KS = 4 * MT;
  auto* y = static_cast<typename Elem<U>::type*>(a.o.y) + b * a.o.sy;
  const Places<MT, NW> pl(a);
  Slab<T, MT, NW> s;
  s.fetch(a, pl, b, k0, kend);
  for (int64_t k = k0; k < kend; k += CK) {
    s.put(pl, Xs);
    __syncthreads();
    if (k + CK < kend) s.fetch(a, pl, b, k + CK, kend);
    f64x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f64x4{0, 0, 0, 0};
    float* mine = Xs + (wid * 16 + r16) * LI;
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      const double x = (double)mine[st * 4 + q];
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = __builtin_amdgcn_mfma_f64_16x16x4f64(Q[(i * 16 + r16) * LQ + st * 4 + q], x, acc[i], 0, 0, 0);
    }
    __syncthreads();  // (all columns of Xs are read by their own wave; the barrier orders its lanes)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) mine[i * 16 + q + 4 * g] = (float)acc[i][g];
    __syncthreads();
    auto* yk = y + (a.tall ? k * a.o.ldy : k);
    const int n = (int)min((int64_t)CK, kend - k);
#pragma unroll
    for (int e = 0; e < 4 * MT; ++e)
      if (pl.k[e] < n) Elem<U>::st(yk + pl.out[e], Xs[pl.at[e]]);
    __syncthreads();
  }
}

// ---- both sides at most D = 16 MT <= 128: x [m][n] (m <= n, zeros behind both) and A, which P = b A + c A A replaces, in LDS
template <int T, int MT>
__global__ __launch_bounds__(512) void k_orth_direct(SmallArgs a, Coefs cf) {
  // D + 4 floats between rows: 16 rows at one group of four columns fall into 16 different 16-byte bank groups
  constexpr int D = 16 * MT, L = D + 4, NL = MT * (MT + 1) / 2, NT = (NL + 7) / 8, NX = (MT * MT + 7) / 8;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  float* X = reinterpret_cast<float*>(lds);
  float* A = X + D * L;
  double* S = reinterpret_cast<double*>(A + D * L);
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, q = lane >> 4;
  const int64_t b = blockIdx.x;
  const int n = (int)a.n, rows = (int)a.o.rows, cols = (int)a.o.cols;
  const auto* x = static_cast<const typename Elem<T>::type*>(a.o.x) + b * a.o.sx;
  double sq = 0.0;
  for (int e = tid; e < D * L; e += 512) X[e] = 0.f;
  __syncthreads();
  for (int e = tid; e < rows * cols; e += 512) {
    const int r = e / cols, c = e - r * cols;
    const float v = Elem<T>::ld(x + r * a.o.ldx + c);
    X[a.tall ? c * L + r : r * L + c] = v;
    sq += (double)v * (double)v;
  }
  for (int w = 32; w > 0; w >>= 1) sq += __shfl_xor(sq, w);
  if (lane == 0) S[wid] = sq;
  __syncthreads();
  const double f = 1.0 / (sqrt(((S[0] + S[1]) + (S[2] + S[3])) + ((S[4] + S[5]) + (S[6] + S[7]))) + a.o.eps);
  for (int e = tid; e < D * L; e += 512) X[e] = (float)((double)X[e] * f);
  __syncthreads();
  // four matrix instructions per 16 columns of the contraction: lane group q takes columns 4 q .. 4 q + 3, one per instruction
  auto rows_product = [&](const float* M, int i, int j, int len) {  // rows i of M against rows j of M
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const float *u = M + (i * 16 + r16) * L + 4 * q, *v = M + (j * 16 + r16) * L + 4 * q;
#pragma unroll 4
    for (int s = 0; s < MT; ++s)
      if (16 * s < len) {
        const f32x4 uu = *reinterpret_cast<const f32x4*>(u + 16 * s), vv = *reinterpret_cast<const f32x4*>(v + 16 * s);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(uu[e], vv[e], acc, 0, 0, 0);
      }
    return acc;
  };
  auto store_sym = [&](int i, int j, f32x4 v) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r = i * 16 + 4 * q + g, c = j * 16 + r16;
      A[r * L + c] = v[g];
      if (i != j) A[c * L + r] = v[g];
    }
  };
  const int mt = (a.m + 15) / 16, nt = (n + 15) / 16, nl = mt * (mt + 1) / 2;
  // this wave's tiles of A and P, and of x
  int li[NT], lj[NT], xi[NX], xj[NX];
#pragma unroll
  for (int u = 0; u < NT; ++u) lower_tile(min(wid + 8 * u, nl - 1), &li[u], &lj[u]);
#pragma unroll
  for (int u = 0; u < NX; ++u) {
    xi[u] = (wid + 8 * u) / nt;
    xj[u] = wid + 8 * u - xi[u] * nt;
  }
  for (int t = 0; t < a.o.steps; ++t) {
    const float ca = (float)cf.v[3 * t], cb = (float)cf.v[3 * t + 1], cc = (float)cf.v[3 * t + 2];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int w = wid + 8 * u;
      if (w < nl) {
        const int i = li[u], j = lj[u];
        store_sym(i, j, rows_product(X, i, j, n));
      }
    }
    __syncthreads();
    f32x4 p[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int w = wid + 8 * u;
      if (w < nl) {
        const int i = li[u], j = lj[u];
        p[u] = rows_product(A, i, j, a.m);
#pragma unroll
        for (int g = 0; g < 4; ++g) p[u][g] = cc * p[u][g] + cb * A[(i * 16 + 4 * q + g) * L + j * 16 + r16];
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int w = wid + 8 * u;
      if (w < nl) {
        const int i = li[u], j = lj[u];
        store_sym(i, j, p[u]);
      }
    }
    __syncthreads();
    f32x4 xn[NX];
#pragma unroll
    for (int u = 0; u < NX; ++u) {
      const int w = wid + 8 * u;
      if (w < mt * nt) {
        const int i = xi[u], j = xj[u];
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        const float *pu = A + (i * 16 + r16) * L + 4 * q, *xv = X + 4 * q * L + j * 16 + r16;
#pragma unroll 4
        for (int s = 0; s < MT; ++s)
          if (16 * s < a.m) {
            const f32x4 uu = *reinterpret_cast<const f32x4*>(pu + 16 * s);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(uu[e], xv[(16 * s + e) * L], acc, 0, 0, 0);
          }
#pragma unroll
        for (int g = 0; g < 4; ++g) xn[u][g] = acc[g] + ca * X[(i * 16 + 4 * q + g) * L + j * 16 + r16];
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NX; ++u) {
      const int w = wid + 8 * u;
      if (w < mt * nt) {
        const int i = xi[u], j = xj[u];
#pragma unroll
        for (int g = 0; g < 4; ++g) X[(i * 16 + 4 * q + g) * L + j * 16 + r16] = xn[u][g];
      }
    }
    __syncthreads();
  }
  auto* y = static_cast<typename Elem<T>::type*>(a.o.y) + b * a.o.sy;
  for (int e = tid; e < rows * cols; e += 512) {
    const int r = e / cols, c = e - r * cols;
    Elem<T>::st(y + r * a.o.ldy + c, X[a.tall ? c * L + r : r * L + c]);
  }
}

template <int T, int U, int MT>
__global__ __launch_bounds__(512) void k_orth_small(SmallArgs a, Coefs cf) {
  constexpr int LQ = Tiles<MT>::LQ, R = Tiles<MT>::R;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  double* A = reinterpret_cast<double*>(lds);
  double *P = A + R * LQ, *Q = P + R * LQ, *scal = A + Tiles<MT>::WORK, *red = scal + 2;
  float* Xs = reinterpret_cast<float*>(red + Tiles<MT>::NL * 256);
  const int64_t b = blockIdx.x;
  gram_range<T, MT, 8>(a, b, 0, a.n, Xs, A, red);
  steps<MT>(a, cf, red, A, P, Q, scal);
  apply_range<T, U, MT, 8>(a, b, 0, a.n, Xs, Q);
}
template <int T, int MT>
__global__ __launch_bounds__(256) void k_orth_gram(SmallArgs a) {
  constexpr int NL = Tiles<MT>::NL, LI = Tiles<MT>::LI;
  __shared__ float Xs[64 * LI];
  __shared__ double part[4 * NL * 256];
  const int64_t b = blockIdx.y, chunks = (a.n + 63) / 64, per = (chunks + a.slices - 1) / a.slices;
  const int64_t k0 = (int64_t)blockIdx.x * per * 64, kend = min(a.n, k0 + per * 64);
  gram_range<T, MT, 4>(a, b, k0, max(k0, kend), Xs, part, a.part + (b * a.slices + blockIdx.x) * (NL * 256));
}
// 32 sums per workgroup, 32 threads to each
__global__ __launch_bounds__(1024) void k_orth_gram_sum(const double* __restrict__ part, int slices, int elems, double* __restrict__ out) {
  __shared__ double S[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t b = blockIdx.y;
  const int e = blockIdx.x * 32 + c;
  double s = 0.0;
#pragma unroll 4
  for (int i = g; i < slices; i += 32) s += part[(b * slices + i) * elems + e];
  S[g][c] = s;
  __syncthreads();
  for (int w = 16; w > 0; w >>= 1) {
    if (g < w) S[g][c] += S[g + w][c];
    __syncthreads();
  }
  if (g == 0) out[b * elems + e] = S[0][c];
}
template <int MT>
__global__ __launch_bounds__(512) void k_orth_steps(SmallArgs a, Coefs cf) {
  constexpr int LQ = Tiles<MT>::LQ, R = Tiles<MT>::R, NL = Tiles<MT>::NL;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  double* A = reinterpret_cast<double*>(lds);
  double *P = A + R * LQ, *Q = P + R * LQ, *scal = Q + R * LQ;
  const int64_t b = blockIdx.x;
  steps<MT>(a, cf, a.gram + b * NL * 256, A, P, Q, scal);
  for (int e = threadIdx.x; e < R * R; e += 512) a.Q[b * R * R + e] = Q[(e / R) * LQ + e % R];
}
template <int T, int U, int MT>
__global__ __launch_bounds__(256) void k_orth_apply(SmallArgs a) {
  constexpr int LQ = Tiles<MT>::LQ, R = Tiles<MT>::R, LI = Tiles<MT>::LI;
  __shared__ double Q[R * LQ];
  __shared__ float Xs[64 * LI];
  const int64_t b = blockIdx.y, chunks = (a.n + 63) / 64, per = (chunks + gridDim.x - 1) / gridDim.x;
  for (int e = threadIdx.x; e < R * R; e += 256) Q[(e / R) * LQ + e % R] = a.Q[b * R * R + e];
  const int64_t k0 = (int64_t)blockIdx.x * per * 64, kend = min(a.n, k0 + per * 64);
  apply_range<T, U, MT, 4>(a, b, k0, kend, Xs, Q);  // (its first barrier orders Q too)
}

namespace {
template <int T, int U, int MT>
int run_small(Ctx* ctx, hipStream_t st, const SmallArgs& a, const Coefs& cf) {
  constexpr int R = Tiles<MT>::R, LQ = Tiles<MT>::LQ, LI = Tiles<MT>::LI, NL = Tiles<MT>::NL;
  constexpr int LDS_STEPS = (3 * R * LQ + 2) * 8, LDS_ALL = (Tiles<MT>::WORK + 2 + NL * 256) * 8 + 128 * LI * 4;
  const unsigned batch = (unsigned)a.o.batch;
  if (a.slices == 1) {
    if (LDS_ALL > 65536) SCL_TRY(ensure_dyn_lds(ctx, reinterpret_cast<const void*>(k_orth_small<T, U, MT>), LDS_ALL));
    SCL_RUN(ctx, k_orth_small<T, U, MT>, dim3(batch), dim3(512), LDS_ALL, st, a, cf);
  } else {
    if (LDS_STEPS > 65536) SCL_TRY(ensure_dyn_lds(ctx, reinterpret_cast<const void*>(k_orth_steps<MT>), LDS_STEPS));
    SCL_RUN(ctx, k_orth_gram<T, MT>, dim3((unsigned)a.slices, batch), dim3(256), 0, st, a);
    SCL_RUN(ctx, k_orth_gram_sum, dim3(NL * 8, batch), dim3(1024), 0, st, a.part, a.slices, NL * 256, a.gram);
    SCL_RUN(ctx, k_orth_steps<MT>, dim3(batch), dim3(512), LDS_STEPS, st, a, cf);
    const int64_t chunks = (a.n + 63) / 64, per = std::max<int64_t>(1, chunks * batch / 768);
    SCL_RUN(ctx, k_orth_apply<T, U, MT>, dim3((unsigned)((chunks + per - 1) / per), batch), dim3(256), 0, st, a);
  }
  return SCLENS_OK;
}
template <int T, int MT>
int run_direct(Ctx* ctx, hipStream_t st, const SmallArgs& a, const Coefs& cf) {
  constexpr int LDS = 2 * 16 * MT * (16 * MT + 4) * 4 + 64;
  if (LDS > 65536) SCL_TRY(ensure_dyn_lds(ctx, reinterpret_cast<const void*>(k_orth_direct<T, MT>), LDS));
  SCL_RUN(ctx, k_orth_direct<T, MT>, dim3((unsigned)a.o.batch), dim3(512), LDS, st, a, cf);
  return SCLENS_OK;
}
template <int T>
int run_direct_t(Ctx* ctx, hipStream_t st, const SmallArgs& a, const Coefs& cf) {
  if (a.n <= 16) return run_direct<T, 1>(ctx, st, a, cf);
  if (a.n <= 32) return run_direct<T, 2>(ctx, st, a, cf);
  if (a.n <= 48) return run_direct<T, 3>(ctx, st, a, cf);
  if (a.n <= 64) return run_direct<T, 4>(ctx, st, a, cf);
  if (a.n <= 96) return run_direct<T, 6>(ctx, st, a, cf);
  return run_direct<T, 8>(ctx, st, a, cf);
}
template <int T, int U>
int run_small_t(Ctx* ctx, hipStream_t st, const SmallArgs& a, const Coefs& cf) {
  if (a.m <= 16) return run_small<T, U, 1>(ctx, st, a, cf);
  if (a.m <= 32) return run_small<T, U, 2>(ctx, st, a, cf);
  if (a.m <= 48) return run_small<T, U, 3>(ctx, st, a, cf);
  return run_small<T, U, 4>(ctx, st, a, cf);
}
// from the caller's type or fp32 (between two runs) to either
int run_small_types(Ctx* ctx, hipStream_t st, const SmallArgs& a, const Coefs& cf, int from, int to) {
  if (from == D_F32 && to == D_F32) return run_small_t<D_F32, D_F32>(ctx, st, a, cf);
  if (from == D_F32) return to == D_BF16 ? run_small_t<D_F32, D_BF16>(ctx, st, a, cf) : run_small_t<D_F32, D_F16>(ctx, st, a, cf);
  if (from == D_BF16) return to == D_F32 ? run_small_t<D_BF16, D_F32>(ctx, st, a, cf) : run_small_t<D_BF16, D_BF16>(ctx, st, a, cf);
  return to == D_F32 ? run_small_t<D_F16, D_F32>(ctx, st, a, cf) : run_small_t<D_F16, D_F16>(ctx, st, a, cf);
}
}  // namespace

// largest |a + b l + c l^2| over 0 <= l <= L
static double largest_quadratic(double a, double b, double c, double L) {
  double v = std::max(std::fabs(a), std::fabs(a + (b + c * L) * L));
  if (c != 0.0) {
    const double l = -b / (2 * c);
    if (l > 0 && l < L) v = std::max(v, std::fabs(a + (b + c * l) * l));
  }
  return v;
}
// The steps from `first` on that one run may take, singular values of at most *bound before and after. What A is off by, m half steps of fp64 of
// bound^2 from every step's rounding, must not pass 2^-8 before the last of them. A step takes an eigenvalue l to l q(l)^2,
// q(l) = a + b l + c l^2, and an error there to q(l) (a + 3 b l + 5 c l^2) times itself (outside the eigenvalues' range, next to zero, to q(l)^2).
// Low-rank matrices on which this was tried in fp64: where the bound is 1e-3 (eleven steps of 3.4445, -4.7750, 2.0315) the result is off by
// 3e-9, at 8e4 (18 steps) by 5e3, then infinite. One step is the definition and always fits.
static int orth_run(const OrthArgs& o, int first, double* bound) {
  const double rounding = (double)std::min(o.rows, o.cols) * 0x1p-53;
  double err = rounding * *bound * *bound;
  int n = 0;
  while (first + n < o.steps && n < MAX_RIDE && (n == 0 || err < 0x1p-8)) {
    const double* c = o.coef + 3 * (first + n);
    const double L = *bound * *bound, q = largest_quadratic(c[0], c[1], c[2], L), dp = largest_quadratic(c[0], 3 * c[1], 5 * c[2], L);
    *bound = orth_step_bound(c[0], c[1], c[2], *bound);
    err = err * q * std::max(q, dp) + rounding * *bound * *bound;
    ++n;
  }
  return n;
}

static bool orth_is_direct(const OrthArgs& o) { return std::max(o.rows, o.cols) <= 128 && o.steps <= MAX_RIDE; }
bool orth_is_small(const OrthArgs& o) {
  return std::max(o.ldx, o.ldy) < ((int64_t)1 << 25) && (orth_is_direct(o) || std::min(o.rows, o.cols) <= 64);
}

int orth_small(Ctx* ctx, hipStream_t st, const OrthArgs& o, void* ws, int64_t ws_bytes, int64_t* need) {
  SmallArgs a{};
  a.o = o;
  a.o.coef = nullptr;
  a.tall = o.rows > o.cols;
  a.m = (int)std::min(o.rows, o.cols);
  a.n = std::max(o.rows, o.cols);
  a.start = 1;
  const int MT = (a.m + 15) / 16, elems = MT * (MT + 1) / 2 * 256;
  const bool direct = orth_is_direct(o);
  if (direct || a.n <= 1024 || o.batch >= 128) a.slices = 1;
  else a.slices = (int)std::max<int64_t>(2, std::min<int64_t>((a.n + 255) / 256, 512 / o.batch));
  double bound = 1.0;
  int run = direct ? o.steps : orth_run(o, 0, &bound);
  Carve c(ws);
  if (a.slices > 1) {
    a.part = c.take<double>(o.batch * a.slices * elems);
    a.gram = c.take<double>(o.batch * elems);
    a.Q = c.take<double>(o.batch * 256 * MT * MT);
  }
  float* between = run < o.steps ? c.take<float>(o.batch * o.rows * o.cols) : nullptr;
  *need = c.used;
  if (c.used > ws_bytes) return ctx->fail(SCLENS_ERR_WORKSPACE, "this call needs " + std::to_string(c.used) + " bytes of device workspace");
  Coefs cf{};
  if (direct) {
    for (int i = 0; i < 3 * o.steps; ++i) cf.v[i] = o.coef[i];
    if (o.dtype == D_F32) return run_direct_t<D_F32>(ctx, st, a, cf);
    if (o.dtype == D_BF16) return run_direct_t<D_BF16>(ctx, st, a, cf);
    return run_direct_t<D_F16>(ctx, st, a, cf);
  }
  for (int first = 0; first < o.steps;) {
    const bool last = first + run == o.steps;
    if (first > 0) {
      a.start = 0;
      a.o.x = between;
      a.o.ldx = o.cols;
      a.o.sx = o.rows * o.cols;
    }
    a.o.y = last ? o.y : between;
    a.o.ldy = last ? o.ldy : o.cols;
    a.o.sy = last ? o.sy : o.rows * o.cols;
    a.o.steps = run;
    for (int i = 0; i < 3 * run; ++i) cf.v[i] = o.coef[3 * first + i];
    SCL_TRY(run_small_types(ctx, st, a, cf, first > 0 ? D_F32 : o.dtype, last ? o.dtype : D_F32));
    first += run;
    run = orth_run(o, first, &bound);
  }
  return SCLENS_OK;
}

}  // namespace scl
