// Products of the dense operators: C[b] = epilogue(alpha * A[b] B[b]') from 16-bit operand images with the contraction contiguous, on
// v_mfma_f32_32x32x16_{bf16,f16} with fp32 accumulation.
//   * fp32 operands come as three bf16 planes (24 bits, exact): six products per term, smallest first -- p2 p0, p0 p2, p1 p1, p1 p0,
//     p0 p1, p0 p0; what is left out (2 p1 p2) is at most 2^-23 of the term and 2^-26 in the mean square, the size of fp32's own rounding.
//   * a workgroup owns one BM x BN tile; both operands go to LDS 64 columns at a time straight from memory (16 bytes per lane), two
//     stages in turn. Chunk q (8 columns) of row r sits in slot q ^ ((r >> 1) & 7): the 32 rows a matrix instruction reads at one
//     column fall into 16 bank groups, two lanes each, which is the rate of a 16-byte read.
//   * the stage loop is a software pipeline of four units (16 columns each): the reads of the next unit are in flight while the
//     matrix instructions of this one run, the copies of the next stage are spread over them, one barrier per stage.
//   * the epilogue turns the accumulators through LDS so that bias, residual, pre-activation and result move 16 bytes per lane along
//     the rows; it can also store the transpose and the mirrored half of a symmetric result.
#include <algorithm>

#include "dense_dev.h"

namespace scl {

typedef __attribute__((address_space(1))) const void glb_cv;
typedef __attribute__((address_space(3))) void lds_v;

// what a lane whose columns lie behind the end of the contraction copies instead
__device__ __attribute__((aligned(16))) unsigned short g_zero_chunk[8] = {0, 0, 0, 0, 0, 0, 0, 0};

struct ProdArgs {
  Product p;
  int tiles_m, tiles_n;  // symmetric: tiles_m (tiles_m + 1) / 2 tiles
  int ksplit;            // slices of the contraction (grid.z), each `kchunk` stages
  int kchunk;
  int nkt;  // stages of one plane pair
};

// XCD-aware order: workgroups go to the 8 XCDs in turn, so consecutive ids are dealt out in 8 contiguous runs of tiles -- the tiles
// that share operand rows then share an L2
__device__ __forceinline__ int xcd_order(int id, int n) {
  const int x = id & 7, q = n >> 3, r = n & 7;
  return x * q + (x < r ? x : r) + (id >> 3);
}

template <int OT, int RT, bool PART>
struct Epilogue {
  // 8 columns from col of row `row`, n of them inside (images with `pad`: all 8, those outside as zeros)
  static __device__ __forceinline__ void apply(const Product& p, int64_t b, int64_t row, int64_t col, int nin, bool row_in, float v[8],
                                               const float* bias8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * p.alpha + bias8[e];
    if (p.pre.p && row_in) store8<OT>(p.pre, b * p.pre.batch + row * p.pre.ld + col, nin, v);
    if (p.act != ACT_NONE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = act_apply(v[e], p.act);
    }
    if (p.res.p && row_in && nin > 0) {
      float r[8];
      load8<RT>(p.res, b * p.res.batch + row * p.res.ld + col, nin, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += p.beta * r[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!row_in || e >= nin) v[e] = 0.f;  // (padding of an image; anything else outside is not stored)
  }
};

// an fp32 product term by term in fp32: only for results that came out NaN, which the pieces also give where an infinity meets a piece
// that is zero (inf * 1.0 contains inf * p1(1.0) = inf * 0)
__device__ __forceinline__ float recompute_f32(const unsigned short* A, const unsigned short* B, int64_t planeA, int64_t planeB, int64_t K) {
  float s = 0.f;
  for (int64_t k = 0; k < K; ++k) {
    const float a = (bf16_to_f32(A[k]) + bf16_to_f32(A[k + planeA])) + bf16_to_f32(A[k + 2 * planeA]);
    const float b = (bf16_to_f32(B[k]) + bf16_to_f32(B[k + planeB])) + bf16_to_f32(B[k + 2 * planeB]);
    s = fmaf(a, b, s);
  }
  return s;
}

template <int MT, int OT, int RT, bool PART, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_product(ProdArgs g) {
  constexpr int NW = WM * WN, BM = WM * TM * 32, BN = WN * TN * 32;
  constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW, NP = PA + PB;  // 1 KB copies (8 rows x 64 columns) per wave and stage
  constexpr int OPA = BM * 128, STAGE = (BM + BN) * 128;
  constexpr bool PL = (MT == D_PL3);
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const Product& p = g.p;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int wm = wid / WN, wn = wid % WN, l31 = lane & 31, h = lane >> 5;

  // ---- the tile
  int ti, tj;
  const int ntiles = (int)gridDim.x;
  const int id = xcd_order((int)blockIdx.x, ntiles);
  if (p.symmetric) {
    int i = (int)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= id) ++i;
    while (i * (i + 1) / 2 > id) --i;
    ti = i;
    tj = id - i * (i + 1) / 2;
  } else {  // bands of 8 tile rows, columns outermost inside a band
    const int band = id / (8 * g.tiles_n), first = band * 8;
    const int rows = min(8, g.tiles_m - first), in = id - band * 8 * g.tiles_n;
    ti = first + in % rows;
    tj = in / rows;
  }
  const int64_t m0 = (int64_t)ti * BM, n0 = (int64_t)tj * BN, batch = blockIdx.y;

  // ---- sources of this wave's copies
  const int srow = lane >> 3, sq = lane & 7;
  const unsigned short* src[NP];
  int chunk8[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const bool isA = i < PA;
    const int r = (isA ? wid * PA + i : wid * PB + i - PA) * 8 + srow;
    const int chunk = sq ^ ((r >> 1) & 7);
    const Mat& m = isA ? p.A : p.B;
    int64_t row = (isA ? m0 : n0) + r;
    const int64_t last = (isA ? p.M : p.N) - 1;
    if (row > last) row = last;  // (its products are not stored)
    src[i] = static_cast<const unsigned short*>(m.p) + batch * m.batch + row * m.ld + 8 * chunk;
    chunk8[i] = 8 * chunk;
  }

  // ---- stages of this slice: stage t = (plane pair t / nkt, columns 64 (t % nkt) ..)
  const int ntot = (PL ? 6 : 1) * g.nkt;
  const int t0 = (int)blockIdx.z * g.kchunk, t1 = min(ntot, t0 + g.kchunk);
  int ld_t = t0;                             // the stage the copies load
  int ld_seg = PL ? t0 / max(1, g.nkt) : 0;  // its plane pair and column block
  int ld_k = t0 - ld_seg * g.nkt;
  int64_t offA = 0, offB = 0;
  auto set_off = [&]() {
    offA = offB = (int64_t)ld_k * 64;
    if (PL) {
      // (A plane, B plane), smallest products first: 20 02 11 10 01 00
      const int pa = (0x001102 >> (4 * ld_seg)) & 15, pb = (0x010120 >> (4 * ld_seg)) & 15;
      offA += pa * p.A.plane;
      offB += pb * p.B.plane;
    }
  };
  auto advance = [&]() {  // past the last stage the copies repeat it; nobody reads the repetition
    if (ld_t + 1 < t1) {
      ++ld_t;
      if (++ld_k == g.nkt) {
        ld_k = 0;
        ++ld_seg;
      }
      set_off();
    }
  };
  auto copy = [&](int buf, int i) {
    const bool isA = i < PA;
    unsigned char* dst = lds + buf * STAGE + (isA ? (wid * PA + i) * 1024 : OPA + (wid * PB + i - PA) * 1024);
    const unsigned short* s = src[i] + (isA ? offA : offB);
    if ((int64_t)ld_k * 64 + chunk8[i] >= p.K) s = g_zero_chunk;
    __builtin_amdgcn_global_load_lds((glb_cv*)s, (lds_v*)dst, 16, 0, 0);
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  int ra[TM], sa[TM], rb[TN], sb[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int r = wm * TM * 32 + i * 32 + l31;
    ra[i] = r * 128;
    sa[i] = (r >> 1) & 7;
  }
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int r = wn * TN * 32 + j * 32 + l31;
    rb[j] = OPA + r * 128;
    sb[j] = (r >> 1) & 7;
  }
  u16x8 av[2][TM], bv[2][TN];
  auto reads = [&](int set, const unsigned char* S, int kk) {
    const int c = 2 * kk + h;
#pragma unroll
    for (int i = 0; i < TM; ++i) av[set][i] = *reinterpret_cast<const u16x8*>(S + ra[i] + ((c ^ sa[i]) << 4));
#pragma unroll
    for (int j = 0; j < TN; ++j) bv[set][j] = *reinterpret_cast<const u16x8*>(S + rb[j] + ((c ^ sb[j]) << 4));
  };
  auto unit = [&](int set, auto pre, auto next) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      pre(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        if constexpr (MT == D_F16)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, av[set][i]), __builtin_bit_cast(f16x8, bv[set][j]),
                                                             acc[i][j], 0, 0, 0);
        else
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, av[set][i]),
                                                              __builtin_bit_cast(bf16x8, bv[set][j]), acc[i][j], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (i == 0) {
        next();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto none = [](int) {};
  // copies 0 .. H-1 of a stage go out in the last unit of the stage before the previous one, H .. NP-1 in the first unit of the previous
  constexpr int H = NP / 2, Q = (H + TM - 1) / TM;
  if (t1 > t0) {
    set_off();
#pragma unroll
    for (int i = 0; i < NP; ++i) copy(0, i);
    __syncthreads();
    advance();
#pragma unroll
    for (int i = 0; i < H; ++i) copy(1, i);
    reads(0, lds, 0);
    for (int t = t0; t < t1; ++t) {
      const int cur = (t - t0) & 1;
      const unsigned char* S = lds + cur * STAGE;
      const unsigned char* Sn = lds + (cur ^ 1) * STAGE;
      unit(0,
           [&](int i) {
#pragma unroll
             for (int q = 0; q < Q; ++q)
               if (H + i * Q + q < NP) copy(cur ^ 1, H + i * Q + q);
           },
           [&]() { reads(1, S, 1); });
      unit(1, none, [&]() { reads(0, S, 2); });
      unit(0, none, [&]() { reads(1, S, 3); });
      __syncthreads();  // every wave has its reads of `cur` behind it; the next stage has landed in the other buffer
      advance();
      unit(1,
           [&](int i) {
#pragma unroll
             for (int q = 0; q < Q; ++q)
               if (i * Q + q < H) copy(cur, i * Q + q);
           },
           [&]() { reads(0, Sn, 0); });
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy may land in the epilogue's LDS
    __syncthreads();
  }

  // ---- epilogue: 32 rows x 32 TN columns of the wave at a time. D: column = lane & 31, row = (e & 3) + 8 (e >> 2) + 4 (lane >> 5)
  constexpr int C = 32 * TN, LP = C + 4, CH = C / 8, RP = 64 / CH;  // RP rows per pass, 8 columns per lane
  float* T = reinterpret_cast<float*>(lds) + wid * 32 * LP;
  const int cc = (lane % CH) * 8, cr = lane / CH;
  const int64_t col = n0 + wn * C + cc;
  const int nin = (int)max((int64_t)0, min((int64_t)8, p.N - col));
  float bias8[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) bias8[e] = 0.f;
  if constexpr (!PART && OT != D_PL3) {
    if (p.bias) {
      typedef typename Elem<OT>::type E;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < nin) bias8[e] = Elem<OT>::ld(static_cast<const E*>(p.bias) + col + e);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) T[((e & 3) + 8 * (e >> 2) + 4 * h) * LP + j * 32 + l31] = acc[i][j][e];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int64_t row0 = m0 + wm * TM * 32 + i * 32;
#pragma unroll
    for (int s = 0; s < 32 / RP; ++s) {
      const int lr = s * RP + cr;
      const int64_t row = row0 + lr;
      float v[8];
      const f32x4 va = *reinterpret_cast<const f32x4*>(&T[lr * LP + cc]), vb = *reinterpret_cast<const f32x4*>(&T[lr * LP + cc + 4]);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = va[e]; v[4 + e] = vb[e]; }
      if constexpr (PART) {
        float* out = p.slabs + (((int64_t)blockIdx.z * p.batch + batch) * p.M + row) * round_up8(p.N) + col;
        if (row < p.M && nin > 0) {
          *reinterpret_cast<f32x4*>(out) = va;
          *reinterpret_cast<f32x4*>(out + 4) = vb;
        }
      } else {
        const bool row_in = row < p.M;
        if constexpr (PL) {
          if (row_in) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (v[e] != v[e] && e < nin)
                v[e] = recompute_f32(static_cast<const unsigned short*>(p.A.p) + batch * p.A.batch + row * p.A.ld,
                                     static_cast<const unsigned short*>(p.B.p) + batch * p.B.batch + (col + e) * p.B.ld, p.A.plane,
                                     p.B.plane, p.K);
          }
        }
        Epilogue<OT, RT, PART>::apply(p, batch, row, col, nin, row_in, v, bias8);
        if (p.out.p) {
          const int n = p.out.pad ? (nin > 0 ? 8 : 0) : nin;
          const bool rin = p.out.pad ? row < round_up8(p.M) : row_in;
          if (rin && n > 0) store8<OT>(p.out, batch * p.out.batch + row * p.out.ld + col, n, v);
        }
        if (p.outT.p || p.symmetric) {
          f32x4 wa = {v[0], v[1], v[2], v[3]}, wb = {v[4], v[5], v[6], v[7]};
          *reinterpret_cast<f32x4*>(&T[lr * LP + cc]) = wa;
          *reinterpret_cast<f32x4*>(&T[lr * LP + cc + 4]) = wb;
        }
      }
    }
    if constexpr (!PART) {
      if (p.outT.p || (p.symmetric && ti != tj)) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const Mat& o = p.symmetric ? p.out : p.outT;
        // column c of the block becomes row n0 + c of the transpose: 8 of its 32 entries per lane
#pragma unroll
        for (int s = 0; s < C / 16; ++s) {
          const int gq = lane & 3, c = s * 16 + (lane >> 2);
          const int64_t trow = n0 + wn * C + c, tcol = row0 + 8 * gq;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = T[(8 * gq + e) * LP + c];
          const int tin = (int)max((int64_t)0, min((int64_t)8, p.M - tcol));
          const int n = o.pad ? (tin > 0 ? 8 : 0) : tin;
          const bool rin = o.pad ? trow < round_up8(p.N) : trow < p.N;
          if (rin && n > 0) store8<OT>(o, batch * o.batch + trow * o.ld + tcol, n, v);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// the slabs of a split contraction, added in order, through the same epilogue: a 32 x 64 block of C per workgroup
template <int OT, int RT, bool PL>
__global__ __launch_bounds__(256) void k_product_join(ProdArgs g) {
  const Product& p = g.p;
  __shared__ float T[32][68];
  const int tid = threadIdx.x, cc = (tid & 7) * 8, lr = tid >> 3;
  const int64_t nb = (p.N + 63) / 64;
  const int64_t row0 = (int64_t)(blockIdx.x / nb) * 32, col0 = (int64_t)(blockIdx.x % nb) * 64, batch = blockIdx.y;
  if (p.symmetric && col0 > row0 + 31) return;  // (every pair below the diagonal is in a block that stays)
  const int64_t row = row0 + lr, col = col0 + cc;
  const int nin = (int)max((int64_t)0, min((int64_t)8, p.N - col));
  const bool row_in = row < p.M;
  float v[8], bias8[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = bias8[e] = 0.f;
  if (row_in && nin > 0) {
    for (int s = 0; s < g.ksplit; ++s) {
      const float* q = p.slabs + (((int64_t)s * p.batch + batch) * p.M + row) * round_up8(p.N) + col;
      const f32x4 a = *reinterpret_cast<const f32x4*>(q), b = *reinterpret_cast<const f32x4*>(q + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] += a[e]; v[4 + e] += b[e]; }
    }
    if constexpr (PL) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v[e] != v[e] && e < nin)
          v[e] = recompute_f32(static_cast<const unsigned short*>(p.A.p) + batch * p.A.batch + row * p.A.ld,
                               static_cast<const unsigned short*>(p.B.p) + batch * p.B.batch + (col + e) * p.B.ld, p.A.plane, p.B.plane, p.K);
    }
    if constexpr (OT != D_PL3) {
      if (p.bias) {
        typedef typename Elem<OT>::type E;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < nin) bias8[e] = Elem<OT>::ld(static_cast<const E*>(p.bias) + col + e);
      }
    }
  }
  Epilogue<OT, RT, false>::apply(p, batch, row, col, nin, row_in, v, bias8);
  if (p.out.p) {
    const int n = p.out.pad ? (nin > 0 ? 8 : 0) : nin;
    const bool rin = p.out.pad ? row < round_up8(p.M) : row_in;
    if (rin && n > 0) store8<OT>(p.out, batch * p.out.batch + row * p.out.ld + col, n, v);  // (a block on the diagonal is whole: both halves)
  }
  if (p.outT.p || p.symmetric) {
#pragma unroll
    for (int e = 0; e < 8; ++e) T[lr][cc + e] = v[e];
    __syncthreads();
    const Mat& o = p.symmetric ? p.out : p.outT;
    const int gq = tid & 3, c = tid >> 2;
    const int64_t trow = col0 + c, tcol = row0 + 8 * gq;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = T[8 * gq + e][c];
    const int tin = (int)max((int64_t)0, min((int64_t)8, p.M - tcol));
    const int n = o.pad ? (tin > 0 ? 8 : 0) : tin;
    const bool rin = o.pad ? trow < round_up8(p.N) : trow < p.N;
    // symmetric: the mirrored copy of what lies below the diagonal only (a block that crosses it wrote both halves above)
    const bool mirror = !p.symmetric || col0 + 63 < row0;
    if (rin && n > 0 && mirror) store8<OT>(o, batch * o.batch + trow * o.ld + tcol, n, v);
  }
}

namespace {

struct Tile { int bm, bn; };
// what a workgroup's tile costs per 64 columns of the contraction, in units of 1e-9 s at full occupancy (measured, see product())
struct Plan { int tile, ksplit, kchunk, tm, tn; int64_t tiles; };

Plan plan_product(int64_t M, int64_t N, int64_t K, int batch, int type, int symmetric, bool may_split) {
  static const int BM[3] = {256, 128, 64};
  const int64_t nst = std::max<int64_t>(1, (type == D_PL3 ? 6 : 1) * ((K + 63) / 64));
  Plan best{};
  double best_t = 1e300;
  for (int t = 0; t < 3; ++t) {
    const int64_t tm = (M + BM[t] - 1) / BM[t], tn = (N + BM[t] - 1) / BM[t];
    const int64_t tiles = (symmetric ? tm * (tm + 1) / 2 : tm * tn) * batch;
    // time of one stage of one workgroup when its CU is full, and workgroups a CU holds at once
    static const double stage_us[3] = {0.95, 0.36, 0.14};
    static const int res[3] = {1, 2, 4};
    for (int ks = 1; ks <= 32; ks *= 2) {
      if (ks > 1 && (!may_split || nst / ks < 4)) break;
      const int64_t kc = (nst + ks - 1) / ks, wg = tiles * ks, slots = 256 * res[t];
      const int64_t rounds = (wg + slots - 1) / slots;
      // an unfull last round: a CU with fewer workgroups than it can hold runs each of them faster
      const int64_t in_last = wg - (rounds - 1) * slots, per_cu = (in_last + 255) / 256;
      double us = ((rounds - 1) * res[t] + per_cu) * (stage_us[t] * kc) + 3.0;
      if (ks > 1) us += 4.0 + (double)ks * M * N * batch * 8.0 / 4e6;
      if (us < best_t) {
        best_t = us;
        best.tile = t;
        best.ksplit = ks;
        best.kchunk = (int)kc;
        best.tm = (int)tm;
        best.tn = (int)tn;
        best.tiles = tiles / batch;
      }
    }
  }
  best.ksplit = (int)((nst + best.kchunk - 1) / best.kchunk);
  return best;
}

template <int MT, int OT, int RT, bool PART, int WM, int WN, int TM, int TN>
int launch(Ctx* ctx, hipStream_t st, const ProdArgs& g, dim3 grid) {
  constexpr int LDS = 2 * (WM * TM + WN * TN) * 32 * 128;
  const void* fn = reinterpret_cast<const void*>(k_product<MT, OT, RT, PART, WM, WN, TM, TN>);
  if (LDS > 65536) SCL_TRY(ensure_dyn_lds(ctx, fn, LDS));
  hipLaunchKernelGGL((k_product<MT, OT, RT, PART, WM, WN, TM, TN>), grid, dim3(WM * WN * 64), LDS, st, g);
  SCL_HIP(ctx, hipGetLastError());
  return SCLENS_OK;
}
template <int MT, int OT, int RT, bool PART>
int launch_tile(Ctx* ctx, hipStream_t st, const ProdArgs& g, dim3 grid, int tile) {
  if (tile == 0) return launch<MT, OT, RT, PART, 2, 4, 4, 2>(ctx, st, g, grid);
  if (tile == 1) return launch<MT, OT, RT, PART, 2, 2, 2, 2>(ctx, st, g, grid);
  return launch<MT, OT, RT, PART, 2, 2, 1, 1>(ctx, st, g, grid);
}
template <int MT, int OT, int RT>
int launch_types(Ctx* ctx, hipStream_t st, const ProdArgs& g, const Plan& pl) {
  const dim3 grid((unsigned)pl.tiles, (unsigned)g.p.batch, (unsigned)pl.ksplit);
  if (pl.ksplit == 1) return launch_tile<MT, OT, RT, false>(ctx, st, g, grid, pl.tile);
  SCL_TRY((launch_tile<MT, D_F32, D_F32, true>(ctx, st, g, grid, pl.tile)));
  const int64_t blocks = ((g.p.M + 31) / 32) * ((g.p.N + 63) / 64);
  hipLaunchKernelGGL((k_product_join<OT, RT, MT == D_PL3>), dim3((unsigned)blocks, (unsigned)g.p.batch), dim3(256), 0, st, g);
  SCL_HIP(ctx, hipGetLastError());
  return SCLENS_OK;
}

}  // namespace

int64_t product_slab_bytes(int64_t M, int64_t N, int64_t K, int batch, int type, int symmetric) {
  const Plan pl = plan_product(M, N, K, batch, type, symmetric, true);
  return pl.ksplit > 1 ? (int64_t)pl.ksplit * batch * M * round_up8(N) * 4 : 0;
}

int product(Ctx* ctx, hipStream_t st, const Product& p) {
  if (p.M <= 0 || p.N <= 0 || p.batch <= 0) return SCLENS_OK;
  const int64_t slab = p.slabs ? product_slab_bytes(p.M, p.N, p.K, p.batch, p.type, p.symmetric) : 0;
  const Plan pl = plan_product(p.M, p.N, p.K, p.batch, p.type, p.symmetric, p.slabs && slab <= p.slab_bytes);
  if (pl.tiles > 0x7fffffff || p.batch > 65535) return ctx->fail(SCLENS_ERR_ARG, "product: too many tiles");
  ProdArgs g{};
  g.p = p;
  g.tiles_m = pl.tm;
  g.tiles_n = pl.tn;
  g.ksplit = pl.ksplit;
  g.kchunk = pl.kchunk;
  g.nkt = (int)((p.K + 63) / 64);
  if (p.type == D_F16) {
    if (p.out_type == D_F16) return launch_types<D_F16, D_F16, D_F16>(ctx, st, g, pl);
    if (p.out_type == D_BF16) return launch_types<D_F16, D_BF16, D_F16>(ctx, st, g, pl);
  } else if (p.type == D_BF16) {
    if (p.out_type == D_BF16) return launch_types<D_BF16, D_BF16, D_BF16>(ctx, st, g, pl);
  } else if (p.type == D_PL3) {
    if (p.out_type == D_PL3) return launch_types<D_PL3, D_PL3, D_PL3>(ctx, st, g, pl);
    if (p.out_type == D_F32 && p.res_type == D_PL3) return launch_types<D_PL3, D_F32, D_PL3>(ctx, st, g, pl);
    if (p.out_type == D_F32) return launch_types<D_PL3, D_F32, D_F32>(ctx, st, g, pl);
  }
  return ctx->fail(SCLENS_ERR_ARG, "product: element types");
}

int product_join(Ctx* ctx, hipStream_t st, const Product& p, int slices) {
  ProdArgs g{};
  g.p = p;
  g.ksplit = slices;
  const dim3 grid((unsigned)(((p.M + 31) / 32) * ((p.N + 63) / 64)), (unsigned)p.batch), blk(256);
  if (p.out_type == D_F32) hipLaunchKernelGGL((k_product_join<D_F32, D_F32, false>), grid, blk, 0, st, g);
  else if (p.out_type == D_BF16) hipLaunchKernelGGL((k_product_join<D_BF16, D_BF16, false>), grid, blk, 0, st, g);
  else hipLaunchKernelGGL((k_product_join<D_F16, D_F16, false>), grid, blk, 0, st, g);
  SCL_HIP(ctx, hipGetLastError());
  return SCLENS_OK;
}

// ------------------------------------------------------------------ images
// 64 rows x 64 columns of the image per workgroup. Straight: 8 columns per lane. Transposed: through LDS, reads along the source's rows.
template <int T, bool TRANS>
__global__ __launch_bounds__(256) void k_pack(const typename Elem<T>::type* __restrict__ src, int64_t ld, int64_t rows, int64_t K, int src_vec,
                                              Mat img) {
  constexpr int IT = T == D_F32 ? D_PL3 : T;
  typedef typename Elem<T>::type E;
  const int64_t r0 = (int64_t)blockIdx.y * 64, k0 = (int64_t)blockIdx.x * 64;
  const int tid = threadIdx.x;
  Mat s;
  s.p = const_cast<E*>(src);
  s.vec = src_vec;
  if constexpr (!TRANS) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = r0 + i * 32 + (tid >> 3), k = k0 + (tid & 7) * 8;
      if (r >= rows) continue;
      float v[8];
      const int n = (int)max((int64_t)0, min((int64_t)8, K - k));
      if (n == 8 && !src_vec) {
        if constexpr (T == D_F32) {
          const f32x8_any a = *reinterpret_cast<const f32x8_any*>(src + r * ld + k);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = a.v[e];
        } else {
          const u16x8_any a = *reinterpret_cast<const u16x8_any*>(src + r * ld + k);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = Elem<T>::ld(&a.v[e]);
        }
      } else
        load8<T>(s, r * ld + k, n, v);
      store8<IT>(img, r * img.ld + k, 8, v);
    }
  } else {
    __shared__ float L[64][65];
    const int c = tid & 63;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t k = k0 + i * 4 + (tid >> 6), r = r0 + c;
      L[i * 4 + (tid >> 6)][c] = (k < K && r < rows) ? Elem<T>::ld(src + k * ld + r) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int lr = i * 32 + (tid >> 3), lk = (tid & 7) * 8;
      if (r0 + lr >= rows) continue;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = L[lk + e][lr];
      store8<IT>(img, (r0 + lr) * img.ld + k0 + lk, 8, v);
    }
  }
}

int pack_image(Ctx* ctx, hipStream_t st, int dtype, const void* src, int64_t ld, bool transposed, int64_t rows, int64_t K, Mat* img) {
  // img->p, plane are the caller's; the leading dimension is that of an image
  img->ld = image_ld(K);
  img->vec = img->pad = 1;
  if (rows <= 0) return SCLENS_OK;
  const int64_t kb = img->ld / 64, rb = (rows + 63) / 64;
  const int size = dtype == D_F32 ? 4 : 2;
  const int vec = !transposed && ld % 8 == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0;
  for (int64_t y0 = 0; y0 < rb; y0 += 65535) {  // grid.y holds 65535 blocks
    const int64_t nb = std::min<int64_t>(65535, rb - y0);
    const dim3 grid((unsigned)kb, (unsigned)nb), block(256);
    const char* s = static_cast<const char*>(src) + (transposed ? y0 * 64 : y0 * 64 * ld) * size;
    Mat m = *img;
    m.p = static_cast<unsigned short*>(img->p) + y0 * 64 * img->ld;
    const int64_t nr = std::min<int64_t>(rows - y0 * 64, nb * 64);
#define SCL_PACK(T)                                                                                                                     if (transposed)                                                                                                                         hipLaunchKernelGGL((k_pack<T, true>), grid, block, 0, st, reinterpret_cast<const Elem<T>::type*>(s), ld, nr, K, vec, m);            else                                                                                                                                    hipLaunchKernelGGL((k_pack<T, false>), grid, block, 0, st, reinterpret_cast<const Elem<T>::type*>(s), ld, nr, K, vec, m);
    if (dtype == D_F32) { SCL_PACK(D_F32) } else if (dtype == D_BF16) { SCL_PACK(D_BF16) } else { SCL_PACK(D_F16) }
#undef SCL_PACK
  }
  SCL_HIP(ctx, hipGetLastError());
  return SCLENS_OK;
}

}  // namespace scl
