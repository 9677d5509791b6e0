// Products of the dense operators: C[b] = epilogue(alpha * A[b] B[b]') on the matrix cores with fp32 accumulation.
//   * 16-bit operands: v_mfma_f32_16x16x32_{bf16,f16}. fp32: v_mfma_f32_32x32x2_f32, or three bf16 planes (24 bits, exact) and six
//     products per term, smallest first -- p2 p0, p0 p2, p1 p1, p1 p0, p0 p1, p0 p0; what is left out (2 p1 p2) is at most 2^-23 of the
//     term and 2^-26 in the mean square, the size of fp32's own rounding. dense_ops.hip has the rule; 4096^3 takes 650 us in planes, their
//     writing included, and about 900 on the fp32 instructions.
//   * an operand lies in memory with the contraction contiguous, or across it (Mat::across: a gradient's transposed operands), and is
//     read as it lies: no transposed copy is written. Rows that do not start on 16 bytes come as a padded copy (k_pack).
//   * a workgroup of four waves owns one BM x BN tile; both operands go to LDS 64 columns at a time (fp32: 32) straight from memory (16
//     bytes per lane), SA and SB stages in turn: three and two (all of LDS) with 128 x 128 per wave or with two workgroups per CU, four
//     where a single workgroup of a small tile would wait for each stage (0.57 us per stage of a 64 x 64 tile with two, whatever the work
//     in it). Chunk q (8 columns) of row r sits in slot q ^ ((r >> 1) & 7): 16 rows at one chunk fall into 16 different 16-byte bank
//     groups, so a 16-byte read runs without conflicts. Rows across the contraction are read with the transposing LDS reads (pair_swz).
//   * the stage loop is a software pipeline of units of 32 columns (fp32: 8): the reads of the next unit and the copies of the stages to
//     come are issued one at a time in the shadow of the matrix instructions, with one barrier a stage.
//   * the epilogue turns the accumulators through LDS so that bias, residual, pre-activation and result move 16 bytes per lane along
//     the rows; it can also store the transpose and the mirrored half of a symmetric result.
// What bounds it: power. 8192^3 in bf16 with SiLU and residual takes 764 us (1.44 PFLOP/s; a plain library product without them 670 to
// 750): the clock is brought down to 1.8 to 2.0 GHz, the matrix cores work in 73 % of the cycles. 16 x 16 x 32 matrix instructions take less of it than 32 x 32 x 16 (below);
// fewer instructions beside them and a barrier with little to wait for came to more than that (860 us before all three). One round of 256 tiles
// (2048 x 2048 -> 8192 with GELU, 66 us) spends 15 us in the launch, the first stages and the epilogue, which nothing overlaps: the
// accumulators leave room for one wave per SIMD. No LDS bank conflicts (counted).
#include <algorithm>
#include <type_traits>

#include "dense_dev.h"

namespace scl {

typedef __attribute__((address_space(1))) const void glb_cv;
typedef __attribute__((address_space(3))) void lds_v;

// the wave's own copies but the N youngest have landed and its LDS reads are done; then everybody's
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

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

template <int N, int I = 0, class F>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    static_for<N, I + 1>(f);
  }
}

// LDS traffic between the lanes of one wave, in order
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int OT, int RT>
struct Epilogue {
  // 8 columns from col of row `row`, n of them inside (images with `pad`: all 8, those outside as zeros)
  static __device__ __forceinline__ void apply(const Product& p, float alpha, int64_t b, int64_t row, int64_t col, int nin, bool row_in,
                                               float v[8], const float* bias8, const Raw8<RT>& res) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * alpha + bias8[e];
    if (p.pre.p && row_in) store8<OT>(p.pre, b * p.pre.batch + row * p.pre.ld + col, nin, v);
    if (p.act != ACT_NONE) act8<false>(v, p.act);
    if (p.res.p && row_in && nin > 0) {
      float r[8];
      res.get(r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += p.beta * r[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!row_in || e >= nin) v[e] = 0.f;  // (padding of an image; anything else outside is not stored)
  }
};

// an fp32 product term by term in fp32: only for results that came out NaN, which the pieces also give where an infinity meets a piece
// that is zero (inf * 1.0 contains inf * p1(1.0) = inf * 0). Eight terms per step, whose loads are on their way together (an image's rows are whole
// chunks, zeros behind K): term by term each waited for its own, and one such result of a long contraction took seconds.
__device__ __forceinline__ float recompute_f32(const unsigned short* A, const unsigned short* B, int64_t planeA, int64_t planeB, int64_t K) {
  auto load = [](const unsigned short* p) { return *reinterpret_cast<const u16x8*>(p); };
  float s = 0.f;
  for (int64_t k = 0; k < K && s == s; k += 8) {
    const u16x8 a0 = load(A + k), a1 = load(A + k + planeA), a2 = load(A + k + 2 * planeA);
    const u16x8 b0 = load(B + k), b1 = load(B + k + planeB), b2 = load(B + k + 2 * planeB);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      s = fmaf((bf16_to_f32(a0[e]) + bf16_to_f32(a1[e])) + bf16_to_f32(a2[e]), (bf16_to_f32(b0[e]) + bf16_to_f32(b1[e])) + bf16_to_f32(b2[e]), s);
  }
  return s;
}

// rows of W elements across the contraction: the 32-byte pair of chunks that column k keeps in place of pair u is u ^ pair_swz(k). The
// columns 4 apart or less and 8 apart that one transposing read touches (k & 3, k & 8) then lie in different banks (256 bytes).
template <int W>
__device__ __forceinline__ int pair_swz(int k) {
  return W % 128 == 0 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2);
}
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
// (__restrict: the inlined call then carries the alias information without which the compiler lets every such read wait for all copies
// to LDS that are on their way)
__device__ __forceinline__ s16x4 read_tr(lds_s16x4* __restrict p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }
template <int ROW>
__device__ __forceinline__ u16x8 read_across(const unsigned char* p) {
  const s16x4 a = read_tr((lds_s16x4*)(p)), b = read_tr((lds_s16x4*)(p + 4 * ROW));
  return __builtin_bit_cast(u16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <int ROW>
__device__ __forceinline__ u16x8 read_words(const unsigned char* p) {
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float*>(p + e * ROW);
  return __builtin_bit_cast(u16x8, v);
}

template <int MT, int OT, int RT, bool PART, bool AC, bool BC, int WM, int WN, int TM, int TN, int SA, int SB>
__global__ __launch_bounds__(WM* WN * 64, TM * TN >= 9 ? 1 : 2) void k_product(ProdArgs g) {
  constexpr int NW = WM * WN, BM = WM * TM * 32, BN = WN * TN * 32;
  constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW, NP = PA + PB;  // 1 KB copies (8 rows x 64 columns) per wave and stage
  static_assert(SA >= SB && SB >= 2, "the first copies go stage by stage");
  constexpr int STA = BM * 128, STB = BN * 128, OPB = SA * STA;  // bytes of a stage's operands; B's stages lie behind A's
  constexpr bool PL = (MT == D_PL3), F32 = (MT == D_F32);
  constexpr int ES = F32 ? 4 : 2, CE = 16 / ES, SC = 128 / ES;  // bytes of an element, elements of a chunk, columns of a stage
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const Product& p = g.p;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid / WN, wn = wid % WN;

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

  // ---- sources of this wave's copies: a uniform base that moves along the contraction, and each lane's place below it (the plan
  // keeps it below 2^32 bytes). A lane's 16 bytes of copy i land at byte 1024 i' + 16 lane of the operand's stage:
  //   rows along the contraction (AC / BC false): row r, slot q of 8 chunks, columns 8 (q ^ ((r >> 1) & 7)) ..
  //   rows across it (true): column k of the contraction, slot of its chunks; in 16 bits the 32-byte pair it is in is swizzled by k
  //   (pair_swz)
  const int srow = lane >> 3, sq = lane & 7;
  const char* baseA = static_cast<const char*>(p.A.p) + ES * (batch * p.A.batch + (AC ? m0 : m0 * p.A.ld));
  const char* baseB = static_cast<const char*>(p.B.p) + ES * (batch * p.B.batch + (BC ? n0 : n0 * p.B.ld));
  const int64_t stepA = AC ? 128 * p.A.ld : 128, stepB = BC ? 128 * p.B.ld : 128;  // bytes per stage
  // ktail != 0: the last stage of the contraction, of which only ktail columns exist: the others are copied from the stage's first
  // chunk / first column (in bounds whatever the matrix) and overwritten with zeros in LDS when they have landed
  auto place = [&](int i, int ktail) -> unsigned {
    const bool isA = i < PA;
    const int grp = isA ? wid * PA + i : wid * PB + i - PA;
    const int64_t rows = isA ? p.M - m0 : p.N - n0, ld = isA ? p.A.ld : p.B.ld;
    if (isA ? AC : BC) {
      const int W = isA ? BM : BN, byte = grp * 1024 + lane * 16;
      int k = byte / (ES * W);
      const int slot = (byte - k * ES * W) >> 4;
      const int c = F32 ? slot : ((slot >> 1) ^ (W == 256 || W == 128 ? pair_swz<256>(k) : pair_swz<64>(k))) * 2 + (slot & 1);
      if (ktail && k >= ktail) k = 0;
      return (unsigned)(ES * (k * ld + (CE * c < rows ? CE * c : 0)));  // (columns behind the end are not stored)
    }
    const int r = grp * 8 + srow;
    int chunk = sq ^ ((r >> 1) & 7);
    if (ktail && CE * chunk >= ktail) chunk = 0;
    const int64_t row = r < rows ? r : rows - 1;  // (products of rows behind the end are not stored)
    return (unsigned)(ES * (row * ld + CE * chunk));
  };
  unsigned voff[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) voff[i] = place(i, 0);

  // ---- stages of this slice: stage t = (plane pair t / nkt, stage t % nkt of the contraction)
  const int ntot = (PL ? 6 : 1) * g.nkt;
  const int t0 = (int)blockIdx.z * g.kchunk, t1 = min(ntot, t0 + g.kchunk);
  const int ktail = (int)(p.K % SC);
  // What the copies of an operand load next: `left` more stages follow one step apart, the last of them stage t; behind it the tail, the
  // next plane, or nothing: then the last stage is copied again and nobody reads the copy.
  struct Ahead {
    int t, left;
    const char* cur;
    int tail;
  };
  auto place_at = [&](Ahead& n, int t, auto is_a) {
    constexpr bool isA = decltype(is_a)::value;
    const int seg = PL ? t / g.nkt : 0, k = t - seg * g.nkt;
    n.cur = (isA ? baseA : baseB) + k * (isA ? stepA : stepB);
    if (PL)  // (A plane, B plane), smallest products first: 20 02 11 10 01 00
      n.cur += 2 * ((isA ? 0x001102 : 0x010120) >> (4 * seg) & 15) * (isA ? p.A.plane : p.B.plane);
    n.left = max(0, min(g.nkt - (ktail != 0 ? 2 : 1) - k, t1 - 1 - t));
    n.t = t + n.left;
    const int tail = ktail != 0 && k + 1 == g.nkt ? ktail : 0;
    if (tail != n.tail) {
      n.tail = tail;
#pragma unroll
      for (int i = isA ? 0 : PA; i < (isA ? PA : NP); ++i) voff[i] = place(i, tail);
    }
  };
  auto advance = [&](Ahead& n, auto is_a) {
    n.cur += decltype(is_a)::value ? stepA : stepB;
    if (--n.left < 0) place_at(n, min(n.t + 1, t1 - 1), is_a);
  };
  Ahead nA = {}, nB = {};
  auto copy = [&](int at, int i) {  // copy i of the stage that lies at `at`
    const bool isA = i < PA;
    unsigned char* dst = lds + at + (isA ? wid * PA + i : wid * PB + i - PA) * 1024;
    __builtin_amdgcn_global_load_lds((glb_cv*)((isA ? nA.cur : nB.cur) + voff[i]), (lds_v*)dst, 16, 0, 0);
  };
  auto zero_tail = [&](int atA, int atB) {
    auto zero = [&](unsigned char* o, auto across, auto w) {
      constexpr int W = decltype(w)::value;
      if constexpr (decltype(across)::value) {  // whole columns of the contraction
        for (int e = ktail * W * ES + tid * 16; e < SC * W * ES; e += NW * 64 * 16) *reinterpret_cast<u16x8*>(o + e) = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
      } else {
        const int first = (ktail + CE - 1) / CE, n = 8 - first;
        for (int e = tid; e < W * n; e += NW * 64) {
          const int r = e / n, c = first + e % n;
          *reinterpret_cast<u16x8*>(o + r * 128 + ((c ^ ((r >> 1) & 7)) << 4)) = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        }
      }
    };
    zero(lds + atA, std::integral_constant<bool, AC>(), std::integral_constant<int, BM>());
    zero(lds + atB, std::integral_constant<bool, BC>(), std::integral_constant<int, BN>());
    wait_lds_barrier();
  };

  // 16 bits: 16 x 16 x 32 tiles, AM x AN of them per wave. Their rate is that of 32 x 32 x 16, with half the traffic of the accumulators and
  // the power that it takes, and power is what holds the clock down: both operands from registers on the whole chip 1.81 PFLOP/s with
  // 32 x 32 x 16, 2.06 with 16 x 16 x 32 if the second operand stays from one instruction to the next, 1.72 if the first one does (random
  // bf16; 2.46 each on zeros). fp32 (156 TFLOP/s either way): 32 x 32 x 2, which has fewer of them.
  constexpr int TS = F32 ? 32 : 16, AM = TM * 32 / TS, AN = TN * 32 / TS, KU = F32 ? 8 : 32, NU = SC / KU;  // KU columns a unit, NU units a stage
  typedef std::conditional_t<F32, f32x16, f32x4> Acc;
  Acc acc[AM][AN] = {};

  // A fragment of TS rows x KU columns: lane (row lr, 16 bytes of columns from chunk NU-th .. on: 2 kk + h, 4 kk + kq). Rows along the
  // contraction: 16 bytes, and rows 16 apart have the same swizzle. Rows across it: two transposing reads of 4 columns each -- 16 lanes name
  // 4 columns x 16 rows (lane i: column i >> 2, rows 4 (i & 3) ..) and lane i receives row i of all four; the four sixteens take columns
  // 8 kq ...
  const int lr = lane & (TS - 1), kq = lane / TS, sw = (lr >> 1) & 7;
  const int ra = (wm * TM * 32 + lr) * 128, rb = (wn * TN * 32 + lr) * 128;
  // fp32: the chunk of 4 columns 8 kk + 4 h .. of the row, its e-th column in the e-th of four matrix instructions; across, four words.
  const int tk = 8 * kq + ((lane & 15) >> 2);
  // (16 rows further the pair number differs in bits that the swizzle changes: with an exclusive or one address does instead of AM, which the
  // largest tile, its first pair a multiple of 8, has no registers for)
  constexpr bool XOR = AC && BC && !F32 && TM == 4;
  int ca[AC && !XOR ? AM : 1], cb[BC && !XOR ? AN : 1];
  if constexpr (AC) {
#pragma unroll
    for (int i = 0; i < (XOR ? 1 : AM); ++i)
      ca[i] = F32 ? 4 * kq * 4 * BM + (wm * TM * 32 + i * 32 + lr) * 4 : tk * 2 * BM + ((wm * TM * 2 + i) ^ pair_swz<BM>(tk)) * 32 + (lane & 3) * 8;
  }
  if constexpr (BC) {
#pragma unroll
    for (int j = 0; j < (XOR ? 1 : AN); ++j)
      cb[j] = F32 ? 4 * kq * 4 * BN + (wn * TN * 32 + j * 32 + lr) * 4 : tk * 2 * BN + ((wn * TN * 2 + j) ^ pair_swz<BN>(tk)) * 32 + (lane & 3) * 8;
  }
  u16x8 av[2][AM], bv[2][AN];
  struct Stage {  // where a stage's operands lie in LDS
    const unsigned char *A, *B;
    int atA, atB;
  };
  auto fragA = [&](const Stage& s, int kk, int i) {
    if constexpr (XOR) return read_across<2 * BM>(lds + ((s.atA + ca[0]) ^ (i << 5)) + kk * KU * 2 * BM);
    else if constexpr (AC && F32) return read_words<4 * BM>(s.A + ca[i] + kk * KU * 4 * BM);
    else if constexpr (AC) return read_across<2 * BM>(s.A + ca[i] + kk * KU * 2 * BM);
    else return *reinterpret_cast<const u16x8*>(s.A + ra + i * TS * 128 + ((((8 / NU) * kk + kq) ^ sw) << 4));
  };
  auto fragB = [&](const Stage& s, int kk, int j) {
    if constexpr (XOR) return read_across<2 * BN>(lds + ((s.atB + cb[0]) ^ (j << 5)) + kk * KU * 2 * BN);
    else if constexpr (BC && F32) return read_words<4 * BN>(s.B + cb[j] + kk * KU * 4 * BN);
    else if constexpr (BC) return read_across<2 * BN>(s.B + cb[j] + kk * KU * 2 * BN);
    else return *reinterpret_cast<const u16x8*>(s.B + rb + j * TS * 128 + ((((8 / NU) * kk + kq) ^ sw) << 4));
  };
  // A unit's AM + AN reads, while the unit before it works on the other set. In the largest tile the first half of A's fragments has one set
  // only (64 registers fewer than two of everything would be 32 too many): they are read last, each when its row of matrix instructions is done.
  constexpr int ONCE = TM == 4 ? AM / 2 : 0;
  auto read = [&](int set, const Stage& s, int kk, int n) {
    if (n < AN) bv[set][n] = fragB(s, kk, n);
    else if (n < AN + AM - ONCE) av[set][n - AN + ONCE] = fragA(s, kk, n - AN + ONCE);
    else av[0][n - AN - AM + ONCE] = fragA(s, kk, n - AN - AM + ONCE);
  };
  // One matrix instruction at a time, and in its shadow what `beside` issues. (HOLD: the large tiles' accumulators stay in the accumulation
  // registers, and each instruction in its place; left to itself, the compiler moves some of either to and fro. No instruction is emitted.)
  constexpr bool HOLD = TM * TN >= 9;
  auto unit = [&](int set, auto beside) {
#pragma unroll
    for (int e = 0; e < (F32 ? 4 : 1); ++e)
#pragma unroll
      for (int i = 0; i < AM; ++i)
#pragma unroll
        for (int j = 0; j < AN; ++j) {
          if constexpr (F32)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(f32x4, bv[set][j])[e], __builtin_bit_cast(f32x4, av[set][i])[e],
                                                             acc[i][j], 0, 0, 0);
          else if constexpr (MT == D_F16)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, bv[set][j]), __builtin_bit_cast(f16x8, av[i < ONCE ? 0 : set][i]),
                                                               acc[i][j], 0, 0, 0);
          else
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, bv[set][j]),
                                                                __builtin_bit_cast(bf16x8, av[i < ONCE ? 0 : set][i]), acc[i][j], 0, 0, 0);
          if constexpr (HOLD) asm volatile("" : "+a"(acc[i][j]));
          __builtin_amdgcn_sched_barrier(0);
          beside((e * AM + i) * AN + j);
          __builtin_amdgcn_sched_barrier(0);
        }
  };
  // one read beside every second matrix instruction where there are enough of those
  constexpr int NM = AM * AN * (F32 ? 4 : 1), NR = AM + AN, SP = NM >= 2 * NR ? 2 : 1;
  auto reads = [&](int set, const Stage& s, int kk, int m) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int once = n - AN - AM + ONCE;  // >= 0: a fragment of one set
      if (m == (once < 0 ? n * SP : std::max(n * SP, AN * (once + 1)))) read(set, s, kk, n);
    }
  };
  // The barrier of stage t stands in its last unit but one, behind the matrix instruction BAR by which the reads of its last columns are
  // back: every wave has them in registers then, so the stage's buffers are free, and stage t + 1 has landed: of the wave's copies only A's of
  // t + 2 .. t + SA - 1 and B's of t + 2 .. t + SB - 1 are younger. Behind it go the copies of B's t + SB, then those of A's t + SA, `p` matrix
  // instructions behind the barrier; a CU takes one per 16 cycles, and the wave whose copy has to wait issues nothing else. B's come first
  // and closer together: with one stage of B less than of A they are the ones that are waited for.
  static_assert(NM >= NR, "a read beside each matrix instruction");
  constexpr int BAR = std::min(NM - 1, std::max((NR - 1) * SP, ONCE * AN) + 8), TOT = NU * NM;
  constexpr int RB = std::max(1, TOT * 3 / 8 / PB), A0 = PB * RB, RA = std::max(1, (TOT - A0 - 1) / PA);
  static_assert(A0 + (PA - 1) * RA + 1 < TOT, "all copies of a stage before the next barrier");
  auto copies = [&](int atA, int atB, int p) {
#pragma unroll
    for (int i = 0; i < PB; ++i)
      if (p == i * RB + 1 - (RB == 1)) copy(atB, PA + i);
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (p == A0 + i * RA + 1 - (RA == 1)) copy(atA, i);
  };
  // A wave is alone on its SIMD, and every instruction of the loop's own costs the matrix cores 4 cycles that nothing fills: the bookkeeping
  // of a stage is a few scalar additions.
  if (t1 > t0) {
    constexpr std::integral_constant<bool, true> opA{};
    constexpr std::integral_constant<bool, false> opB{};
    place_at(nA, t0, opA);
    place_at(nB, t0, opB);
#pragma unroll
    for (int b = 0; b < SA; ++b) {
      if (b < SB) {
        if (b > 0) advance(nB, opB);
#pragma unroll
        for (int i = PA; i < NP; ++i) copy(OPB + b * STB, i);
      }
      if (b > 0) advance(nA, opA);
#pragma unroll
      for (int i = 0; i < PA; ++i) copy(b * STA, i);
    }
    wait_barrier<(SA - 1) * PA + (SB - 1) * PB>();
    int to_tail = ktail != 0 ? g.nkt - 1 - t0 % g.nkt : 0x7fffffff;  // stages until the next one that ends inside its columns
    if (to_tail == 0) {
      zero_tail(0, OPB);
      to_tail = g.nkt;
    }
#pragma unroll
    for (int n = 0; n < NR; ++n) read(0, Stage{lds, lds + OPB, 0, OPB}, 0, n);
    // where A's and B's stages t, t + 1 .. lie in LDS
    int oa[SA], ob[SB];
#pragma unroll
    for (int i = 0; i < SA; ++i) oa[i] = i * STA;
#pragma unroll
    for (int i = 0; i < SB; ++i) ob[i] = OPB + i * STB;
    for (int t = t0; t < t1; ++t) {
      const Stage now{lds + oa[0], lds + ob[0], oa[0], ob[0]}, next{lds + oa[1], lds + ob[1], oa[1], ob[1]};
#pragma unroll
      for (int u = 0; u < NU; ++u)
        unit(u & 1, [&](int m) {
          if (u + 1 < NU) reads((u & 1) ^ 1, now, u + 1, m);
          else reads(0, next, 0, m);
          // (before this stage's barrier: what is left of the copies behind the last one, whose buffers have moved to the end)
          const int p = (u - (NU - 2)) * NM + m - BAR - 1;
          if (p < 0) copies(oa[SA - 1], ob[SB - 1], p + TOT);
          if (p >= 0) copies(oa[0], ob[0], p);
          if (p == -1) {
            wait_barrier<(SA - 2) * PA + (SB - 2) * PB>();
            if (--to_tail == 0) {
              zero_tail(oa[1], ob[1]);
              to_tail = g.nkt;
            }
            advance(nB, opB);
            advance(nA, opA);
          }
        });
      const int a0 = oa[0], b0 = ob[0];
#pragma unroll
      for (int i = 0; i + 1 < SA; ++i) oa[i] = oa[i + 1];
#pragma unroll
      for (int i = 0; i + 1 < SB; ++i) ob[i] = ob[i + 1];
      oa[SA - 1] = a0;
      ob[SB - 1] = b0;
    }
    wait_barrier<0>();  // no copy may land in the epilogue's LDS
  }
  if constexpr (HOLD) asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");  // (the last results have been written)

  // ---- epilogue: 32 rows x 32 TN columns of the wave at a time, turned through LDS. D (B's rows are the matrix instruction's rows):
  // row of C = lane % TS, column = 4 (lane / TS) + (e & 3), in fp32 + 8 (e >> 2). The loops stay rolled: unrolled, their 250 KB of instructions (every
  // activation, every edge) cost a workgroup 25 us.
  constexpr int C = 32 * TN, LP = C + 4, CH = TN == 3 ? 16 : C / 8, RP = 64 / CH, NS = 32 / RP;  // RP rows per pass, 8 columns per lane
  float* T = reinterpret_cast<float*>(lds) + wid * 32 * LP;
  // (96 columns are twelve lanes of sixteen: the last four repeat the twelfth and store nothing)
  const bool mine = (lane % CH) * 8 < C;
  const int cc = mine ? (lane % CH) * 8 : C - 8, cr = lane / CH;
  const int64_t col = n0 + wn * C + cc, row_w = m0 + wm * TM * 32;
  const int nin = mine ? (int)max((int64_t)0, min((int64_t)8, p.N - col)) : 0;
  auto to_lds = [&](int i) {
    static_for<TM>([&](auto I) {
      constexpr int n = decltype(I)::value;
      if (i == n) {
        // (the two markers keep the branches from being merged into one that picks its accumulators by index, from scratch memory)
        asm volatile("; rows %0" ::"n"(n) : "memory");
#pragma unroll
        for (int j = 0; j < AN; ++j)
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<f32x4*>(&T[lr * LP + j * 32 + 8 * e + 4 * kq]) =
                  f32x4{acc[n][j][4 * e], acc[n][j][4 * e + 1], acc[n][j][4 * e + 2], acc[n][j][4 * e + 3]};
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) *reinterpret_cast<f32x4*>(&T[(16 * e + lr) * LP + j * 16 + 4 * kq]) = acc[2 * n + e][j];
          }
        asm volatile("; rows %0" ::"n"(n) : "memory");
      }
    });
    wave_sync();
  };
  auto from_lds = [&](int lr, float v[8]) {
    const f32x4 va = *reinterpret_cast<const f32x4*>(&T[lr * LP + cc]), vb = *reinterpret_cast<const f32x4*>(&T[lr * LP + cc + 4]);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = va[e]; v[4 + e] = vb[e]; }
  };
  if constexpr (PART) {
    float* out = p.slabs + (((int64_t)blockIdx.z * p.batch + batch) * p.M + row_w) * round_up8(p.N) + col;
#pragma unroll 1
    for (int i = 0; i < TM; ++i) {
      to_lds(i);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        float v[8];
        from_lds(s * RP + cr, v);
        const int64_t r = i * 32 + s * RP + cr;
        if (row_w + r < p.M && nin > 0) {
          *reinterpret_cast<f32x4*>(out + r * round_up8(p.N)) = f32x4{v[0], v[1], v[2], v[3]};
          *reinterpret_cast<f32x4*>(out + r * round_up8(p.N) + 4) = f32x4{v[4], v[5], v[6], v[7]};
        }
      }
      wave_sync();
    }
  } else {
    const float alpha = p.scale ? p.alpha * *p.scale : p.alpha;
    float bias8[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bias8[e] = 0.f;
    if constexpr (OT != D_PL3) {
      if (p.bias) {
        Mat b;
        b.p = const_cast<void*>(p.bias);
        b.vec = reinterpret_cast<uintptr_t>(p.bias) % 16 == 0;  // (col is a multiple of 8)
        load8<OT>(b, col, nin, bias8);
      }
    }
    const Mat& ot = p.symmetric ? p.out : p.outT;
    const bool turned = p.outT.p || (p.symmetric && ti != tj);
    // column c of block i becomes row n0 + c of the transpose: 8 of its 32 entries per lane
    auto turn = [&](int i) {
      if (!turned) return;
      wave_sync();
#pragma unroll 1
      for (int s = 0; s < C / 16; ++s) {
          const int gq = lane & 3, c = s * 16 + (lane >> 2);
          const int64_t trow = n0 + wn * C + c, tcol = row_w + i * 32 + 8 * gq;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = T[(8 * gq + e) * LP + c];
          const int tin = (int)max((int64_t)0, min((int64_t)8, p.M - tcol));
          const int n = ot.pad ? (tin > 0 ? 8 : 0) : tin;
          const bool rin = ot.pad ? trow < round_up8(p.N) : trow < p.N;
          if (rin && n > 0) store8<OT>(ot, batch * ot.batch + trow * ot.ld + tcol, n, v);
        }
      };
    // A tile that lies inside the matrix, all its rows on 16 bytes: nothing to guard. Loads and stores share a counter, so a residual
    // that came through registers would make every pass wait for the stores of the pass before it (32 times a microsecond): it goes to
    // LDS, the next block's while this one is worked on, and only the copies are waited for (the stores since are counted off).
    const bool inside = m0 + BM <= p.M && n0 + BN <= p.N && (!p.out.p || p.out.vec) && (!p.pre.p || p.pre.vec) && (!p.res.p || p.res.vec);
    if constexpr (!PL) {
      if (inside) {
        const int64_t row0 = row_w + cr;
        const char* pr = static_cast<const char*>(p.res.p) + ES * (batch * p.res.batch + row0 * p.res.ld + col);
        constexpr int OS = OT == D_F32 ? 4 : 2, NST = NS * OS / 2;  // 16-byte stores of a block per result
        static_assert(PART || PL || (RT == D_F32 ? 4 : 2) == ES, "the residual has the operands' size");
        char* po = static_cast<char*>(p.out.p) + OS * (batch * p.out.batch + row0 * p.out.ld + col);
        char* pz = static_cast<char*>(p.pre.p) + OS * (batch * p.pre.batch + row0 * p.pre.ld + col);
        const int64_t sr = ES * RP * p.res.ld, so = OS * RP * p.out.ld, sz = OS * RP * p.pre.ld;
        const bool has_res = p.res.p != nullptr, has_out = p.out.p != nullptr, has_pre = p.pre.p != nullptr;
        constexpr int RB = NS * 1024 * ES / 2;  // bytes of a block's residual
        unsigned char* R = lds + NW * 32 * LP * 4 + wid * 2 * RB;
        auto copy_res = [&](int buf) {
#pragma unroll
          for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int q = 0; q < ES / 2; ++q)
              __builtin_amdgcn_global_load_lds((glb_cv*)(pr + 16 * q), (lds_v*)(R + buf * RB + (s * (ES / 2) + q) * 1024), 16, 0, 0);
            pr += sr;
          }
        };
        Mat plain;
        plain.vec = 1;
        if (has_res) copy_res(0);
#pragma unroll 1
        for (int i = 0; i < TM; ++i) {
          if (has_res) {
            if (i == 0 || turned) wait_vm<0>();
            else if (has_out && has_pre) wait_vm<2 * NST>();
            else wait_vm<NST>();
            if (i + 1 < TM) copy_res((i + 1) & 1);
          }
          to_lds(i);
          const unsigned char* Ri = R + (i & 1) * RB + lane * 16;
#pragma unroll 1
          for (int s = 0; s < NS; ++s) {
            float v[8];
            from_lds(s * RP + cr, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(v[e], alpha, bias8[e]);
            if (has_pre) {
              plain.p = pz;
              if (mine) store8<OT>(plain, 0, 8, v);
              pz += sz;
            }
            if (p.act != ACT_NONE) act8<false>(v, p.act);
            if (has_res) {
              Raw8<RT> r;
              float f[8];
#pragma unroll
              for (int q = 0; q < ES / 2; ++q) r.r[q] = *reinterpret_cast<const u16x8*>(Ri + (s * (ES / 2) + q) * 1024);
              r.get(f);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = fmaf(p.beta, f[e], v[e]);
            }
            if (has_out) {
              plain.p = po;
              if (mine) store8<OT>(plain, 0, 8, v);
              po += so;
            }
            if (turned && mine) {
              *reinterpret_cast<f32x4*>(&T[(s * RP + cr) * LP + cc]) = f32x4{v[0], v[1], v[2], v[3]};
              *reinterpret_cast<f32x4*>(&T[(s * RP + cr) * LP + cc + 4]) = f32x4{v[4], v[5], v[6], v[7]};
            }
          }
          turn(i);
          wave_sync();
        }
        return;
      }
    }
#pragma unroll 1
    for (int i = 0; i < TM; ++i) {
      to_lds(i);
#pragma unroll 1
      for (int s = 0; s < NS; ++s) {
        const int lr = s * RP + cr;
        const int64_t row = row_w + i * 32 + lr;
        const bool row_in = row < p.M;
        float v[8];
        from_lds(lr, v);
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
        Raw8<RT> res;
        if (p.res.p && row_in && nin > 0) res.load(p.res, batch * p.res.batch + row * p.res.ld + col, nin);
        Epilogue<OT, RT>::apply(p, alpha, batch, row, col, nin, row_in, v, bias8, res);
        if (p.out.p) {
          const int n = p.out.pad ? (nin > 0 ? 8 : 0) : nin;
          const bool rin = p.out.pad ? row < round_up8(p.M) : row_in;
          if (rin && n > 0) store8<OT>(p.out, batch * p.out.batch + row * p.out.ld + col, n, v);
        }
        if (turned && mine) {
          *reinterpret_cast<f32x4*>(&T[lr * LP + cc]) = f32x4{v[0], v[1], v[2], v[3]};
          *reinterpret_cast<f32x4*>(&T[lr * LP + cc + 4]) = f32x4{v[4], v[5], v[6], v[7]};
        }
      }
      turn(i);
      wave_sync();
    }
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
  const float alpha = p.scale ? p.alpha * *p.scale : p.alpha;
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
  Raw8<RT> res;
  if (p.res.p && row_in && nin > 0) res.load(p.res, batch * p.res.batch + row * p.res.ld + col, nin);
  Epilogue<OT, RT>::apply(p, alpha, batch, row, col, nin, row_in, v, bias8, res);
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

struct Plan { int tile, ksplit, kchunk, tm, tn; int64_t tiles; double us; };

// a lane's place below its tile's base has 32 bits: the small tile's 64 rows (across: a stage's 64 or 32
// columns) have at most MAX_CONTRACTION elements, in fp32 MAX_CONTRACTION_F32, a large tile's 256 at most MAX_LD_BIG
constexpr int64_t MAX_LD_BIG = (int64_t)1 << 22;

struct TileKind {
  int bm;            // the tile is bm x bm
  int per_cu;        // workgroups a CU holds (LDS)
  double stage1_us;  // one stage of a workgroup alone on its CU
  double stage_us;   // one stage of each of per_cu workgroups of a full CU (the whole chip busy: lower clocks)
  double fixed_us;   // launch, first stages, epilogue
};
// measured at 16 and 64 stages on 64 to 1024 tiles
constexpr int NTILES = 5;
const TileKind TILES[NTILES] = {{256, 1, 1.1, 1.30, 15.0},
                                  {192, 1, 0.80, 0.90, 11.0},
                                  {128, 2, 0.73, 1.02, 4.0},
                                  {128, 1, 0.53, 0.55, 6.0},
                                  {64, 2, 0.29, 0.41, 3.5}};
// fp32 on the fp32 matrix cores, stages of 32 columns: bound by the matrix instructions in every tile (workgroups that share a CU take turns),
// so the two smallest do; the larger ones' residual would not fit LDS beside the accumulators. Three stages instead of four let a third
// workgroup of the smallest onto a CU (gradients of 7373 x 480 -> 4838: 733 -> 595 us)
const TileKind TILES_F32[NTILES] = {{0, 1, 0, 0, 0}, {0, 1, 0, 0, 0}, {0, 1, 0, 0, 0}, {128, 1, 2.0, 2.1, 6.0}, {64, 3, 0.55, 1.6, 4.5}};

// The tile and the slices of the contraction with the least time by the figures above: rounds of the chip's 256 CUs, the stages of a
// workgroup, and for slices the slabs written, read and joined by a second launch.
Plan plan_product(int64_t M, int64_t N, int64_t K, int batch, int type, int symmetric, bool may_split) {
  const int64_t nst = std::max<int64_t>(1, type == D_F32 ? (K + 31) / 32 : (type == D_PL3 ? 6 : 1) * ((K + 63) / 64));
  Plan best{};
  double best_t = 1e300;
  for (int t = K > MAX_LD_BIG ? NTILES - 1 : 0; t < NTILES; ++t) {
    const TileKind& k = (type == D_F32 ? TILES_F32 : TILES)[t];
    if (k.bm == 0) continue;
    const int64_t tm = (M + k.bm - 1) / k.bm, tn = (N + k.bm - 1) / k.bm;
    const int64_t tiles = (symmetric ? tm * (tm + 1) / 2 : tm * tn) * batch;
    for (int ks = 1; ks <= 32; ks *= 2) {
      if (ks > 1 && (!may_split || nst / ks < 4)) break;
      const int64_t kc = (nst + ks - 1) / ks, wg = tiles * ks, slots = 256 * k.per_cu, full = wg / slots, rest = wg - full * slots;
      double us = full * (k.stage_us * kc + k.fixed_us);
      if (rest > 0) us += (rest <= 256 ? k.stage1_us : k.stage_us) * kc + k.fixed_us;
      if (ks > 1) us += 3.0 + 0.4 * ks + (double)ks * M * N * batch * (symmetric ? 4.0 : 8.0) / 4e6;
      if (us < best_t) {
        best_t = us;
        best.tile = t;
        best.ksplit = ks;
        best.kchunk = (int)kc;
        best.tm = (int)tm;
        best.tn = (int)tn;
        best.tiles = tiles / batch;
        best.us = us;
      }
    }
  }
  best.ksplit = (int)((nst + best.kchunk - 1) / best.kchunk);
  return best;
}

template <int MT, int OT, int RT, bool PART, bool AC, bool BC, int WM, int WN, int TM, int TN, int SA, int SB>
int launch(Ctx* ctx, hipStream_t st, const ProdArgs& g, dim3 grid) {
  // the stages; the epilogue's block of fp32 and two blocks of the residual per wave
  constexpr int LDS = std::max((SA * WM * TM + SB * WN * TN) * 32 * 128,
                               WM * WN * (32 * (32 * TN + 4) * 4 + 2 * 32 * (TN == 3 ? 128 : 32 * TN) * (MT == D_F32 ? 4 : 2)));
  static_assert(LDS <= 163840, "LDS of a CU");
  const void* fn = reinterpret_cast<const void*>(k_product<MT, OT, RT, PART, AC, BC, WM, WN, TM, TN, SA, SB>);
  if (LDS > 65536) SCL_TRY(ensure_dyn_lds(ctx, fn, LDS));
  SCL_RUN(ctx, k_product<MT, OT, RT, PART, AC, BC, WM, WN, TM, TN, SA, SB>, grid, dim3(WM * WN * 64), LDS, st, g);
  return SCLENS_OK;
}
template <int MT, int OT, int RT, bool PART, bool AC, bool BC>
int launch_tile(Ctx* ctx, hipStream_t st, const ProdArgs& g, dim3 grid, int tile) {
  if constexpr (MT != D_F32) {
    if (tile == 0) return launch<MT, OT, RT, PART, AC, BC, 2, 2, 4, 4, 3, 2>(ctx, st, g, grid);
    if (tile == 1) return launch<MT, OT, RT, PART, AC, BC, 2, 2, 3, 3, 3, 3>(ctx, st, g, grid);
    if (tile == 2) return launch<MT, OT, RT, PART, AC, BC, 2, 2, 2, 2, 3, 2>(ctx, st, g, grid);
  }
  switch (tile) {
    case 3: return launch<MT, OT, RT, PART, AC, BC, 2, 2, 2, 2, 4, 4>(ctx, st, g, grid);
    default: return launch<MT, OT, RT, PART, AC, BC, 2, 2, 1, 1, MT == D_F32 ? 3 : 4, MT == D_F32 ? 3 : 4>(ctx, st, g, grid);
  }
}
template <int MT, int OT, int RT, bool AC = false, bool BC = false>
int launch_types(Ctx* ctx, hipStream_t st, const ProdArgs& g, const Plan& pl) {
  const dim3 grid((unsigned)pl.tiles, (unsigned)g.p.batch, (unsigned)pl.ksplit);
  if (pl.ksplit == 1) return launch_tile<MT, OT, RT, false, AC, BC>(ctx, st, g, grid, pl.tile);
  SCL_TRY((launch_tile<MT, D_F32, D_F32, true, AC, BC>(ctx, st, g, grid, pl.tile)));
  const int64_t blocks = ((g.p.M + 31) / 32) * ((g.p.N + 63) / 64);
  SCL_RUN(ctx, k_product_join<OT, RT, MT == D_PL3>, dim3((unsigned)blocks, (unsigned)g.p.batch), dim3(256), 0, st, g);
  return SCLENS_OK;
}

}  // namespace

int64_t product_slab_bytes(int64_t M, int64_t N, int64_t K, int batch, int type, int symmetric) {
  const Plan pl = plan_product(M, N, K, batch, type, symmetric, true);
  return pl.ksplit > 1 ? (int64_t)pl.ksplit * batch * M * round_up8(N) * 4 : 0;
}

double product_us(int64_t M, int64_t N, int64_t K, int batch, int type, int symmetric) {
  return plan_product(M, N, K, batch, type, symmetric, true).us;
}

int product(Ctx* ctx, hipStream_t st, const Product& p) {
  if (p.M <= 0 || p.N <= 0 || p.batch <= 0) return SCLENS_OK;
  const int64_t slab = p.slabs ? product_slab_bytes(p.M, p.N, p.K, p.batch, p.type, p.symmetric) : 0;
  const Plan pl = plan_product(p.M, p.N, p.K, p.batch, p.type, p.symmetric, p.slabs && slab <= p.slab_bytes);
  for (const Mat* m : {&p.A, &p.B})
    if (m->ld > (p.type == D_F32 && !m->across ? MAX_CONTRACTION_F32 : MAX_CONTRACTION))
      return ctx->fail(SCLENS_ERR_ARG, "product: an operand's rows are too long");
  if (pl.tiles >= 1 << 24 || p.batch > 65535) return ctx->fail(SCLENS_ERR_ARG, "product: too many tiles");
  ProdArgs g{};
  g.p = p;
  g.tiles_m = pl.tm;
  g.tiles_n = pl.tn;
  g.ksplit = pl.ksplit;
  g.kchunk = pl.kchunk;
  g.nkt = (int)(p.type == D_F32 ? (p.K + 31) / 32 : (p.K + 63) / 64);
  const int form = (p.A.across ? 2 : 0) + (p.B.across ? 1 : 0);
  if (p.type == D_F16) {
    if (p.out_type == D_F16) {
      if (form == 0) return launch_types<D_F16, D_F16, D_F16>(ctx, st, g, pl);
      if (form == 1) return launch_types<D_F16, D_F16, D_F16, false, true>(ctx, st, g, pl);
      if (form == 3) return launch_types<D_F16, D_F16, D_F16, true, true>(ctx, st, g, pl);
    }
    if (p.out_type == D_BF16 && form == 0) return launch_types<D_F16, D_BF16, D_F16>(ctx, st, g, pl);
    if (p.out_type == D_BF16 && form == 1) return launch_types<D_F16, D_BF16, D_F16, false, true>(ctx, st, g, pl);
  } else if (p.type == D_BF16 && p.out_type == D_BF16) {
    if (form == 0) return launch_types<D_BF16, D_BF16, D_BF16>(ctx, st, g, pl);
    if (form == 1) return launch_types<D_BF16, D_BF16, D_BF16, false, true>(ctx, st, g, pl);
    if (form == 3) return launch_types<D_BF16, D_BF16, D_BF16, true, true>(ctx, st, g, pl);
  } else if (p.type == D_F32 && p.out_type == D_F32) {
    if (form == 0) return launch_types<D_F32, D_F32, D_F32>(ctx, st, g, pl);
    if (form == 1) return launch_types<D_F32, D_F32, D_F32, false, true>(ctx, st, g, pl);
    if (form == 3) return launch_types<D_F32, D_F32, D_F32, true, true>(ctx, st, g, pl);
  } else if (form == 0) {
    if (p.type == D_PL3 && p.out_type == D_PL3) return launch_types<D_PL3, D_PL3, D_PL3>(ctx, st, g, pl);
    if (p.type == D_PL3 && p.out_type == D_F32 && p.res_type == D_PL3) return launch_types<D_PL3, D_F32, D_PL3>(ctx, st, g, pl);
    if (p.type == D_PL3 && p.out_type == D_F32) return launch_types<D_PL3, D_F32, D_F32>(ctx, st, g, pl);
  }
  return ctx->fail(SCLENS_ERR_ARG, "product: element types");
}

int product_join(Ctx* ctx, hipStream_t st, const Product& p, int slices) {
  ProdArgs g{};
  g.p = p;
  g.ksplit = slices;
  const dim3 grid((unsigned)(((p.M + 31) / 32) * ((p.N + 63) / 64)), (unsigned)p.batch), blk(256);
  if (p.out_type == D_F32) SCL_RUN(ctx, k_product_join<D_F32, D_F32, false>, grid, blk, 0, st, g);
  else if (p.out_type == D_BF16) SCL_RUN(ctx, k_product_join<D_BF16, D_BF16, false>, grid, blk, 0, st, g);
  else SCL_RUN(ctx, k_product_join<D_F16, D_F16, false>, grid, blk, 0, st, g);
  return SCLENS_OK;
}

// ------------------------------------------------------------------ images
// 64 rows x 64 columns of the image per workgroup. Straight: 8 columns per lane. Transposed: through LDS, reads along the source's rows.
// A launch makes one image or two of equal K (the second one's row blocks behind the first one's `blocks`: 1001 columns of 777 and 515
// rows of fp16 take 5.2 us together and 6.6 one after the other).
struct PackSource {
  const void* p;
  int64_t ld, rows;
  int vec;
  Mat img;
};
template <int T, int IT, bool TRANS>
__global__ __launch_bounds__(256) void k_pack(PackSource first, PackSource second, int blocks, int64_t K) {
  typedef typename Elem<T>::type E;
  const bool in_first = (int)blockIdx.y < blocks;
  const PackSource& o = in_first ? first : second;
  const E* __restrict__ src = static_cast<const E*>(o.p);
  const int64_t ld = o.ld, rows = o.rows;
  const int src_vec = o.vec;
  const Mat& img = o.img;
  const int64_t r0 = (int64_t)((int)blockIdx.y - (in_first ? 0 : blocks)) * 64, k0 = (int64_t)blockIdx.x * 64;
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

namespace {
int launch_pack(Ctx* ctx, hipStream_t st, int dtype, int image, bool transposed, const PackSource& first, const PackSource& second, int64_t K) {
  const int64_t n1 = (first.rows + 63) / 64, n2 = (second.rows + 63) / 64;
  const dim3 grid((unsigned)(image_ld(K) / 64), (unsigned)(n1 + n2)), block(256);
#define SCL_PACK(T, I, TR) SCL_RUN(ctx, k_pack<T, I, TR>, grid, block, 0, st, first, second, (int)n1, K)
  if (image == D_PL3 && transposed) SCL_PACK(D_F32, D_PL3, true);
  else if (image == D_PL3) SCL_PACK(D_F32, D_PL3, false);
  else if (transposed) return ctx->fail(SCLENS_ERR_ARG, "pack_image: transposed only into planes");
  else if (dtype == D_F32) SCL_PACK(D_F32, D_F32, false);
  else if (dtype == D_BF16) SCL_PACK(D_BF16, D_BF16, false);
  else SCL_PACK(D_F16, D_F16, false);
#undef SCL_PACK
  return SCLENS_OK;
}
PackSource pack_source(int dtype, const void* src, int64_t ld, bool transposed, int64_t rows, int64_t K, Mat* img) {
  // img->p, plane are the caller's; the leading dimension is that of an image
  img->ld = image_ld(K);
  img->vec = img->pad = 1;
  PackSource s{src, ld, rows, !transposed && ld % 8 == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0, *img};
  return s;
}
constexpr int64_t MAX_PACK_ROWS = (int64_t)65535 * 64;  // grid.y holds 65535 blocks
}  // namespace

int pack_image(Ctx* ctx, hipStream_t st, int dtype, int image, const void* src, int64_t ld, bool transposed, int64_t rows, int64_t K, Mat* img) {
  const PackSource all = pack_source(dtype, src, ld, transposed, rows, K, img);
  const int size = dtype == D_F32 ? 4 : 2;
  for (int64_t r = 0; r < rows; r += MAX_PACK_ROWS) {
    PackSource s = all;
    s.p = static_cast<const char*>(src) + (transposed ? r : r * ld) * size;
    s.rows = std::min(MAX_PACK_ROWS, rows - r);
    s.img.p = static_cast<char*>(img->p) + r * img->ld * (image == D_F32 ? 4 : 2);
    SCL_TRY(launch_pack(ctx, st, dtype, image, transposed, s, PackSource(), K));
  }
  return SCLENS_OK;
}

int pack_pair(Ctx* ctx, hipStream_t st, int dtype, int image, const void* a, int64_t lda, int64_t rows_a, Mat* img_a, const void* b, int64_t ldb,
              int64_t rows_b, Mat* img_b, int64_t K) {
  if (img_a && img_b && rows_a > 0 && rows_b > 0 && rows_a + rows_b + 64 <= MAX_PACK_ROWS)
    return launch_pack(ctx, st, dtype, image, false, pack_source(dtype, a, lda, false, rows_a, K, img_a),
                       pack_source(dtype, b, ldb, false, rows_b, K, img_b), K);
  if (img_a) SCL_TRY(pack_image(ctx, st, dtype, image, a, lda, false, rows_a, K, img_a));
  if (img_b) SCL_TRY(pack_image(ctx, st, dtype, image, b, ldb, false, rows_b, K, img_b));
  return SCLENS_OK;
}
}  // namespace scl
