// Products with one short side: the long operand is streamed once past at most 16 rows (k_rows, any type) or, in fp32 or from rows
// that do not start on 16 bytes, at most 128 rows (k_stream). Both are bound by reading the long operand; the matrix cores (16 x 16 x 32
// tiles, the long operand as the rows of the tile) have room to spare: 26 % of their cycles at 40 short rows in fp32 (six products per
// term). Measured: 4096 x 4096 bf16 weights past one row 7.6 us (4.4 TB/s), fp32 20 000 x 10 000 past 40 rows 182 us (4.4 TB/s; a large
// copy moves 4.9).
#include <algorithm>

#include "dense_dev.h"

namespace scl {

typedef __attribute__((address_space(1))) const void glb_cv;
typedef __attribute__((address_space(3))) void lds_v;

// eight elements k .. k+7 of a row that ends at K, at any element address
template <int T> struct Chunk;
template <> struct Chunk<D_F32> {
  float v[8];
  __device__ __forceinline__ void load(const float* row, int64_t k, int64_t K) {
    if (k + 8 <= K) {
      const f32x8_any a = *reinterpret_cast<const f32x8_any*>(row + k);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = a.v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k + e < K ? row[k + e] : 0.f;
    }
  }
};
template <int T> struct Chunk16 {
  u16x8 v;
  __device__ __forceinline__ void load(const unsigned short* row, int64_t k, int64_t K) {
    if (k + 8 <= K) {
      const u16x8_any a = *reinterpret_cast<const u16x8_any*>(row + k);
      v = __builtin_bit_cast(u16x8, a);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k + e < K ? row[k + e] : 0;
    }
  }
};
template <> struct Chunk<D_BF16> : Chunk16<D_BF16> {};
template <> struct Chunk<D_F16> : Chunk16<D_F16> {};

template <int T>
__device__ __forceinline__ f32x4 mfma16(u16x8 a, u16x8 b, f32x4 c) {
  if constexpr (T == D_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight fp32 values as three bf16 pieces each, without a look at infinities: those (and what would round up to one) leave NaN in the
// second piece, and a result that comes out NaN is formed again in fp32.
__device__ __forceinline__ void split8(const float v[8], u16x8 out[3]) {
  unsigned d[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      const bf16x2 h = {(__bf16)a, (__bf16)b};
      const unsigned w = __builtin_bit_cast(unsigned, h);
      d[p][i] = w;
      if (p < 2) {
        a -= __uint_as_float(w << 16);
        b -= __uint_as_float(w & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int p = 0; p < 3; ++p) __builtin_memcpy(&out[p], d[p], 16);
}

// ---- at most 16 rows of x: 16 rows of w per workgroup, the contraction dealt out to its 8 waves in runs of 128 columns
template <int T>
__global__ __launch_bounds__(512) void k_rows(LinearArgs a) {
  typedef typename Elem<T>::type E;
  __shared__ float S[8][256];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, r16 = lane & 15, q = lane >> 4;
  const int64_t n0 = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 16;
  if (n0 >= a.N) return;
  const E* wr = static_cast<const E*>(a.w) + min(n0 + r16, a.N - 1) * a.ldw;  // (rows behind the end: not stored)
  const E* xr = static_cast<const E*>(a.x) + min((int64_t)r16, a.M - 1) * a.ldx;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int64_t k0 = wid * 128; k0 < a.K; k0 += 8 * 128) {
    Chunk<T> w[4], x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i].load(wr, k0 + 32 * i + 8 * q, a.K);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i].load(xr, k0 + 32 * i + 8 * q, a.K);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (T == D_F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i].v[e], x[i].v[e], acc, 0, 0, 0);
      } else
        acc = mfma16<T>(w[i].v, x[i].v, acc);
    }
  }
  *reinterpret_cast<f32x4*>(&S[wid][lane * 4]) = acc;
  __syncthreads();
  if (tid >= 256) return;
  const int nn = tid & 15;
  const int64_t m = tid >> 4, n = n0 + nn;
  if (m >= a.M || n >= a.N) return;
  const int at = ((nn >> 2) * 16 + (int)m) * 4 + (nn & 3);
  float z = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) z += S[w][at];
  if (a.bias) z += Elem<T>::ld(static_cast<const E*>(a.bias) + n);
  if (a.pre) Elem<T>::st(static_cast<E*>(a.pre) + m * a.ldz + n, z);
  z = act_any<false>(z, a.act);
  if (a.res) z += Elem<T>::ld(static_cast<const E*>(a.res) + m * a.ldr + n);
  Elem<T>::st(static_cast<E*>(a.y) + m * a.ldy + n, z);
}

int linear_rows(Ctx* ctx, hipStream_t st, const LinearArgs& a) {
  const int64_t groups = (a.N + 15) / 16, x = std::min<int64_t>(groups, 1 << 22);  // (a grid's side holds fewer than 2^32 threads)
  const dim3 grid((unsigned)x, (unsigned)((groups + x - 1) / x)), blk(512);
  if (a.dtype == D_F32) SCL_RUN(ctx, k_rows<D_F32>, grid, blk, 0, st, a);
  else if (a.dtype == D_BF16) SCL_RUN(ctx, k_rows<D_BF16>, grid, blk, 0, st, a);
  else SCL_RUN(ctx, k_rows<D_F16>, grid, blk, 0, st, a);
  return SCLENS_OK;
}

// ---- at most 128 short rows (an image: three bf16 planes for fp32): 256 long rows per workgroup, 32 per wave, the contraction cut into
// grid.y slices of whole 64-column stages. The short operand's stages sit in LDS (D in turn, chunk q of row r in slot
// q ^ ((r >> 1) & 7)); the long one goes from memory to registers D stages ahead and, in fp32, is taken apart there. A packed copy of it, which the tiled product would read, costs three times the traffic: fp32 20 000 x 10 000 onto 40 took 949 us
// that way (196 us this way, 205 with the long operand two stages ahead instead of three), bf16 20 001 x 10 001 (rows on 2 bytes) 281 us.
struct StreamArgs {
  const void* big;
  int64_t ldb, R, K;
  Mat small;
  int64_t S;
  float* slabs;       // [slice][M][round_up8(N)]
  int64_t slab;       // elements of a slice
  int64_t sr, ss;     // strides of the long and the short index in a slab
  int kchunk;         // stages per slice
};
// stages that the long operand is fetched ahead: three where the registers hold them
constexpr int stream_depth(int NT) { return NT <= 4 ? 3 : 2; }
template <int T, int NT>
__global__ __launch_bounds__(512, 2) void k_stream(StreamArgs a) {
  typedef typename Elem<T>::type E;
  constexpr int NP = T == D_F32 ? 3 : 1, ROWS = NT * 16;
  constexpr int PLANE = ROWS * 128, STAGE = NP * PLANE, PIECES = STAGE / 1024;
  constexpr int LOADS = T == D_F32 ? 8 : 4, COPIES = PIECES / 8;  // 16-byte loads of a stage's fetch and its copies per wave, at least
  constexpr int D = stream_depth(NT);
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, q = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * 256 + wid * 32;
  const E* rows[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) rows[i] = static_cast<const E*>(a.big) + min(row0 + i * 16 + r16, a.R - 1) * a.ldb;
  const int nst = (int)((a.K + 63) / 64);
  const int t0 = (int)blockIdx.y * a.kchunk, t1 = min(nst, t0 + a.kchunk);
  auto copy = [&](int buf, int t) {
    for (int p = wid; p < PIECES; p += 8) {  // 1 KB: 8 rows x 64 columns of a plane
      const int plane = p / (ROWS / 8), r = (p % (ROWS / 8)) * 8 + (lane >> 3);
      const int c = (lane & 7) ^ ((r >> 1) & 7);  // (an image's rows are whole stages)
      const unsigned short* s = static_cast<const unsigned short*>(a.small.p) + plane * a.small.plane +
                                min((int64_t)r, a.S - 1) * a.small.ld + (int64_t)t * 64 + 8 * c;
      __builtin_amdgcn_global_load_lds((glb_cv*)s, (lds_v*)(lds + buf * STAGE + p * 1024), 16, 0, 0);
    }
  };
  Chunk<T> ahead[D][2][2];
  auto fetch = [&](Chunk<T>(&n)[2][2], int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) n[i][kk].load(rows[i], (int64_t)t * 64 + kk * 32 + q * 8, a.K);
  };
  f32x4 acc[2][NT];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto stage = [&](Chunk<T>(&n)[2][2], int t, int cur) {
    // This stage's copy has landed on all sides; younger ones may still be on their way: with D = 2 the fetch of t + 1, with D = 3 the fetches
    // of t + 1 and t + 2 and the copy between them. (A stage that ends inside its 64 columns is fetched with fewer loads, so they cannot be
    // counted off.)
    if (t + D - 1 < t1 && (int64_t)(t + D) * 64 <= a.K)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((D - 1) * LOADS + (D - 2) * COPIES) : "memory");
    else if (D == 3 && t + 1 < t1 && (int64_t)(t + 2) * 64 <= a.K)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS + COPIES) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    u16x8 A[2][2][NP];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        if constexpr (T == D_F32) split8(n[i][kk].v, A[i][kk]);
        else A[i][kk][0] = n[i][kk].v;
      }
    if (t + D - 1 < t1) copy((cur + D - 1) % D, t + D - 1);
    if (t + D < t1) fetch(n, t + D);
    const unsigned char* B = lds + cur * STAGE;
    // up to four column tiles together, so that six products of one accumulator are not issued one after the other
    constexpr int G = NT <= 4 ? NT : NT / 2;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int j0 = 0; j0 < NT; j0 += G) {
        u16x8 b[G][NP];
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const int r = (j0 + j) * 16 + r16, c = 4 * kk + q;
#pragma unroll
          for (int p = 0; p < NP; ++p) b[j][p] = *reinterpret_cast<const u16x8*>(B + p * PLANE + r * 128 + ((c ^ ((r >> 1) & 7)) << 4));
        }
        auto term = [&](int pa, int pb) {
#pragma unroll
          for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[i][j0 + j] = mfma16<T>(A[i][kk][pa], b[j][pb], acc[i][j0 + j]);
        };
        if constexpr (T == D_F32) {
          term(2, 0);
          term(0, 2);
          term(1, 1);
          term(1, 0);
          term(0, 1);
        }
        term(0, 0);
      }
  };
#pragma unroll
  for (int i = 0; i < D; ++i)
    if (t0 + i < t1) {
      if (i < D - 1) copy(i, t0 + i);
      fetch(ahead[i], t0 + i);
    }
  for (int t = t0; t < t1; t += D) {
#pragma unroll
    for (int i = 0; i < D; ++i)
      if (t + i < t1) stage(ahead[i], t + i, i);
  }
  float* out = a.slabs + (int64_t)blockIdx.y * a.slab;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t s = j * 16 + r16;
      if (s >= a.S) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t r = row0 + i * 16 + 4 * q + e;
        if (r >= a.R) continue;
        float v = acc[i][j][e];
        if (T == D_F32 && v != v) {  // an infinity that met a zero piece, or was taken apart: this slice's terms again in fp32
          const float* x = static_cast<const float*>(a.big) + r * a.ldb;
          const unsigned short* y = static_cast<const unsigned short*>(a.small.p) + s * a.small.ld;
          v = 0.f;
          const int64_t k1 = min(a.K, (int64_t)t1 * 64);
          for (int64_t k = (int64_t)t0 * 64; k < k1 && v == v; ++k)
            v = fmaf(x[k], (bf16_to_f32(y[k]) + bf16_to_f32(y[k + a.small.plane])) + bf16_to_f32(y[k + 2 * a.small.plane]), v);
        }
        out[r * a.sr + s * a.ss] = v;
      }
    }
}

namespace {
template <int T, int NT>
int launch_stream(Ctx* ctx, hipStream_t st, const StreamArgs& a, int slices) {
  constexpr int LDS = stream_depth(NT) * (T == D_F32 ? 3 : 1) * NT * 16 * 128;
  if (LDS > 65536) SCL_TRY(ensure_dyn_lds(ctx, reinterpret_cast<const void*>(k_stream<T, NT>), LDS));
  SCL_RUN(ctx, k_stream<T, NT>, dim3((unsigned)((a.R + 255) / 256), (unsigned)slices), dim3(512), LDS, st, a);
  return SCLENS_OK;
}
template <int T>
int launch_stream_t(Ctx* ctx, hipStream_t st, const StreamArgs& a, int slices) {
  if (a.S <= 16) return launch_stream<T, 1>(ctx, st, a, slices);
  if (a.S <= 32) return launch_stream<T, 2>(ctx, st, a, slices);
  if (a.S <= 48) return launch_stream<T, 3>(ctx, st, a, slices);
  if (a.S <= 64) return launch_stream<T, 4>(ctx, st, a, slices);
  if (a.S <= 96) return launch_stream<T, 6>(ctx, st, a, slices);
  return launch_stream<T, 8>(ctx, st, a, slices);
}
}  // namespace

// The slices with the least time: rounds of the 256 CUs (one workgroup each), 2 us per stage and 6 per workgroup, the slabs written and
// read at 4 TB/s, their join.
int stream_slices(int64_t R, int64_t S, int64_t K, int* kchunk) {
  const int64_t nst = (K + 63) / 64, groups = (R + 255) / 256;
  double best = 1e300;
  int slices = 1;
  for (int64_t s = 1; s <= std::min<int64_t>(nst, 64); ++s) {
    const int64_t kc = (nst + s - 1) / s, n = (nst + kc - 1) / kc;
    const double us = (double)((groups * n + 255) / 256) * (kc * 2.0 + 6.0) + n * (0.4 + (double)R * S * 8.0 / 4e6);
    if (us < best) {
      best = us;
      slices = (int)n;
      *kchunk = (int)kc;
    }
  }
  return slices;
}

// What all of it takes -- the short operand's copy, the stream, the join -- against the tiles' product_us. Within 30 % of 27 measured shapes,
// and on the faster side for 26 of them (fp32 64 x 4096 x 4096: 41 us this way, 31 in tiles; 20 000 x 93 x 10 000: 282 and 512).
double stream_us(int64_t R, int64_t S, int64_t K, int dtype) {
  int kchunk;
  const int64_t n = stream_slices(R, S, K, &kchunk), groups = (R + 255) / 256, nt = (S + 15) / 16;
  const double stage = dtype == D_F32 ? 1.4 + 0.33 * nt : 1.0 + 0.15 * nt;
  return 9.5 + (double)((groups * n + 255) / 256) * (kchunk * stage + 4.0) + n * (0.4 + (double)R * S * 8.0 / 4e6);
}

int stream_product(Ctx* ctx, hipStream_t st, int dtype, const void* big, int64_t ldb, int64_t R, const Mat& small, int64_t S, int64_t K,
                   float* slabs, int64_t slab, int64_t sr, int64_t ss) {
  StreamArgs a{};
  a.big = big; a.ldb = ldb; a.R = R; a.K = K;
  a.small = small; a.S = S;
  a.slabs = slabs; a.slab = slab; a.sr = sr; a.ss = ss;
  const int slices = stream_slices(R, S, K, &a.kchunk);
  if (dtype == D_F32) return launch_stream_t<D_F32>(ctx, st, a, slices);
  if (dtype == D_BF16) return launch_stream_t<D_BF16>(ctx, st, a, slices);
  return launch_stream_t<D_F16>(ctx, st, a, slices);
}

}  // namespace scl
