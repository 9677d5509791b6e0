// Small products and gradients in one launch, for matrices of any address and order: where the tiles would first need packed copies (fp32,
// rows that do not start on 16 bytes) or a gradient several passes, the launches cost more than the work. 32 x 32 results per workgroup,
// a quarter per wave, on v_mfma_f32_16x16x4 (16-bit operands convert exactly); 32 columns of the contraction at a time go through
// registers to LDS, the next 32 on their way meanwhile. What bounds it is the latency of those steps, not the rate: gradients of 200 x 93
// -> 50 in fp32 with ReLU take 9.9 us one after another in a graph, 2.4 and 1.07 for each of dw's seven steps (0.8 without an activation, whose kind
// is decided per element); dx (two steps, 4.6 us alone) and the column sums (5.2 us alone) run beside it.
#include <algorithm>

#include "dense_dev.h"

namespace scl {

// element (r, k) at p[r * ld + k], across: p[k * ld + r]; with z: times act'(z), which lies the same way
struct SmallOperand {
  const void *p, *z;
  int64_t ld, ldz, rows;
  int across;
};

template <int T>
struct SmallLoad {
  float v[4];
  // four elements of a 32 x 32 block: row r, columns k .. k+3, or column k, rows r .. r+3 (across)
  __device__ __forceinline__ void fetch(const SmallOperand& o, int act, int64_t r0, int64_t k0, int64_t K) {
    typedef typename Elem<T>::type E;
    const int a = threadIdx.x >> 3, b = (threadIdx.x & 7) * 4;
    const int64_t r = r0 + (o.across ? b : a), k = k0 + (o.across ? a : b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t re = r + (o.across ? e : 0), ke = k + (o.across ? 0 : e);
      v[e] = 0.f;
      if (re < o.rows && ke < K) {
        v[e] = Elem<T>::ld(static_cast<const E*>(o.p) + (o.across ? ke * o.ld + re : re * o.ld + ke));
        if (o.z) {
          v[e] *= act_any<true>(Elem<T>::ld(static_cast<const E*>(o.z) + (o.across ? ke * o.ldz + re : re * o.ldz + ke)), act);
        }
      }
    }
  }
  __device__ __forceinline__ void put(float* S, int across) const {  // S[r][k], 36 floats between rows
    const int a = threadIdx.x >> 3, b = (threadIdx.x & 7) * 4;
    if (across) {
#pragma unroll
      for (int e = 0; e < 4; ++e) S[(b + e) * 36 + a] = v[e];
    } else
      *reinterpret_cast<f32x4*>(S + a * 36 + b) = f32x4{v[0], v[1], v[2], v[3]};
  }
};

// acc: this wave's 16 x 16 quarter of A B' at (r0, c0): rows 4 q + g, column lane & 15
template <int T>
__device__ __forceinline__ f32x4 small_tile(const SmallOperand& A, const SmallOperand& B, int act, int64_t r0, int64_t c0, int64_t K, float* S) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  SmallLoad<T> a, b;
  if (K > 0) {
    a.fetch(A, act, r0, 0, K);
    b.fetch(B, act, c0, 0, K);
  }
  for (int64_t k = 0; k < K; k += 32) {
    a.put(S, A.across);
    b.put(S + 32 * 36, B.across);
    __syncthreads();
    if (k + 32 < K) {
      a.fetch(A, act, r0, k + 32, K);
      b.fetch(B, act, c0, k + 32, K);
    }
    const float *u = S + ((wid >> 1) * 16 + r16) * 36 + 4 * q, *v = S + (32 + (wid & 1) * 16 + r16) * 36 + 4 * q;
#pragma unroll
    for (int s = 0; s < 2; ++s) {  // columns 16 s + 4 q + e: one of the four per instruction
      const f32x4 uu = *reinterpret_cast<const f32x4*>(u + 16 * s), vv = *reinterpret_cast<const f32x4*>(v + 16 * s);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(uu[e], vv[e], acc, 0, 0, 0);
    }
    __syncthreads();
  }
  return acc;
}

template <int T>
__global__ __launch_bounds__(256) void k_small_linear(LinearArgs a) {
  typedef typename Elem<T>::type E;
  __shared__ __attribute__((aligned(16))) float S[64 * 36];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
  const int64_t nb = (a.N + 31) / 32, m0 = (blockIdx.x / nb) * 32, n0 = (blockIdx.x % nb) * 32;
  const SmallOperand A = {a.x, nullptr, a.ldx, 0, a.M, 0}, B = {a.w, nullptr, a.ldw, 0, a.N, 0};
  const f32x4 acc = small_tile<T>(A, B, ACT_NONE, m0, n0, a.K, S);
  const int64_t n = n0 + (wid & 1) * 16 + r16;
  if (n >= a.N) return;
  const float bias = a.bias ? Elem<T>::ld(static_cast<const E*>(a.bias) + n) : 0.f;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int64_t m = m0 + (wid >> 1) * 16 + 4 * q + g;
    if (m >= a.M) continue;
    float z = acc[g] + bias;
    if (a.pre) Elem<T>::st(static_cast<E*>(a.pre) + m * a.ldz + n, z);
    z = act_any<false>(z, a.act);
    if (a.res) z += Elem<T>::ld(static_cast<const E*>(a.res) + m * a.ldr + n);
    Elem<T>::st(static_cast<E*>(a.y) + m * a.ldy + n, z);
  }
}

// blocks of dx, then of dw, then of db (32 columns each, 8 threads to a column)
template <int T>
__global__ __launch_bounds__(256) void k_small_backward(LinearBwdArgs a, int ndx, int ndw) {
  typedef typename Elem<T>::type E;
  __shared__ __attribute__((aligned(16))) float S[64 * 36];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
  const void* z = a.act == ACT_NONE ? nullptr : a.pre;
  int id = (int)blockIdx.x;
  if (id < ndx + ndw) {
    const bool dx = id < ndx;
    if (!dx) id -= ndx;
    const int64_t rows = dx ? a.M : a.N, kb = (a.K + 31) / 32, r0 = (id / kb) * 32, c0 = (id % kb) * 32;
    const SmallOperand A = {a.dy, z, a.lddy, a.ldz, rows, !dx};
    const SmallOperand B = {dx ? a.w : a.x, nullptr, dx ? a.ldw : a.ldx, 0, a.K, 1};
    const f32x4 acc = small_tile<T>(A, B, a.act, r0, c0, dx ? a.N : a.M, S);
    const int64_t c = c0 + (wid & 1) * 16 + r16, ld = dx ? a.lddx : a.lddw;
    E* out = static_cast<E*>(dx ? a.dx : a.dw);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int64_t r = r0 + (wid >> 1) * 16 + 4 * q + g;
      if (r < rows && c < a.K) Elem<T>::st(out + r * ld + c, acc[g]);
    }
    return;
  }
  id -= ndx + ndw;
  const int c = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int64_t n = (int64_t)id * 32 + c;
  double s = 0.0;
  if (n < a.N)
#pragma unroll 4
    for (int64_t m = part; m < a.M; m += 8) {
      float v = Elem<T>::ld(static_cast<const E*>(a.dy) + m * a.lddy + n);
      if (z) v *= act_any<true>(Elem<T>::ld(static_cast<const E*>(z) + m * a.ldz + n), a.act);
      s += (double)v;
    }
  double* D = reinterpret_cast<double*>(S);
  D[part * 32 + c] = s;
  __syncthreads();
  if (part == 0 && n < a.N) {
    for (int p = 1; p < 8; ++p) s += D[p * 32 + c];
    Elem<T>::st(static_cast<E*>(a.db) + n, (float)s);
  }
}

// Forward: at most 2^28 flops and 1024 columns of the contraction, where the tiles would need packed copies (fp32 300 x 300 -> 300: 7.7 us
// against 20; operands on 16 bytes feed the tiles as they lie). Backward, against up to six launches of 25 to 30 us: at most 2^26 flops a
// product and 384 rows of either contraction (fp32 200 x 93 -> 50: 11 us against 36; 512 x 256 -> 512 would take 27).
bool linear_is_small(const LinearArgs& a) { return a.K <= 1024 && (double)a.M * a.N * a.K <= (double)(1 << 27); }
bool backward_is_small(const LinearBwdArgs& a) { return std::max(a.M, a.N) <= 384 && (double)a.M * a.N * a.K <= (double)(1 << 25); }

int linear_small(Ctx* ctx, hipStream_t st, const LinearArgs& a) {
  const dim3 grid((unsigned)(((a.M + 31) / 32) * ((a.N + 31) / 32))), blk(256);
  if (a.dtype == D_F32) SCL_RUN(ctx, k_small_linear<D_F32>, grid, blk, 0, st, a);
  else if (a.dtype == D_BF16) SCL_RUN(ctx, k_small_linear<D_BF16>, grid, blk, 0, st, a);
  else SCL_RUN(ctx, k_small_linear<D_F16>, grid, blk, 0, st, a);
  return SCLENS_OK;
}
int backward_small(Ctx* ctx, hipStream_t st, const LinearBwdArgs& a) {
  const int64_t kb = (a.K + 31) / 32, ndx = a.dx ? ((a.M + 31) / 32) * kb : 0, ndw = a.dw ? ((a.N + 31) / 32) * kb : 0;
  const int64_t ndb = a.db ? (a.N + 31) / 32 : 0, all = ndx + ndw + ndb;
  if (all == 0) return SCLENS_OK;
  const dim3 grid((unsigned)all), blk(256);
  if (a.dtype == D_F32) SCL_RUN(ctx, k_small_backward<D_F32>, grid, blk, 0, st, a, (int)ndx, (int)ndw);
  else if (a.dtype == D_BF16) SCL_RUN(ctx, k_small_backward<D_BF16>, grid, blk, 0, st, a, (int)ndx, (int)ndw);
  else SCL_RUN(ctx, k_small_backward<D_F16>, grid, blk, 0, st, a, (int)ndx, (int)ndw);
  return SCLENS_OK;
}

}  // namespace scl
