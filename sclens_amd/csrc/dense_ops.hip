// Dense operators on device tensors (sclens_amd/dense.py):
//   linear            y = act(x w' + b) + r
//   linear_backward   dz = dy act'(z),  dx = dz w,  dw = dz' x,  db = column sums of dz
//   orthogonalize     x0 = g / (|g|_F + eps);  per step (a, b, c): A = x x',  x <- a x + (b A + c A A) x
// The products are those of dense_gemm.hip; here are the passes around them and the order of the launches. Every launch goes to the
// caller's stream, scratch is the caller's, nothing synchronises: a call can be captured into a graph.
#include <algorithm>
#include <cmath>

#include "dense_dev.h"

namespace scl {

namespace {
int no_room(Ctx* ctx, int64_t need) {
  return ctx->fail(SCLENS_ERR_WORKSPACE, "this call needs " + std::to_string(need) + " bytes of device workspace");
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// a matrix whose rows start on 16 bytes and are whole 16-byte chunks feeds the products of its own type as it lies
bool direct(int dtype, const void* p, int64_t ld, int64_t K) {
  const int64_t chunk = dtype == D_F32 ? 4 : 8;
  return ld % chunk == 0 && ld <= ((int64_t)1 << (dtype == D_F32 ? 21 : 22)) && K % chunk == 0 && aligned16(p);
}

Mat user_mat(const void* p, int64_t ld, int64_t batch = 0) {
  Mat m;
  m.p = const_cast<void*>(p);
  m.ld = ld;
  m.batch = batch;
  m.vec = ld % 8 == 0 && batch % 8 == 0 && aligned16(p);
  return m;
}
Mat image_of(Carve& c, int image, int64_t rows, int64_t K, int64_t batch = 1) {
  Mat m;
  m.batch = image_elems(rows, K);
  m.plane = m.batch * batch;
  m.ld = image_ld(K);
  m.vec = m.pad = 1;
  m.p = image == D_F32 ? static_cast<void*>(c.take<float>(m.plane)) : c.take<unsigned short>(m.plane * (image == D_PL3 ? 3 : 1));
  return m;
}
// fp32 products: on the fp32 matrix cores as the matrices lie, or from three bf16 planes each at 1.5 times the rate, which first have to
// be written (4 bytes read, 6 written per element and operand, 4 TB/s)
bool planes_pay(int64_t M, int64_t N, int64_t K, int64_t packed_elems, int batch = 1, int symmetric = 0) {
  return product_us(M, N, K, batch, D_PL3, symmetric) + (double)packed_elems * 10.0 / 4e6 + 6.0 < product_us(M, N, K, batch, D_F32, symmetric);
}
}  // namespace

// ------------------------------------------------------------------ linear
// One short side: at most 16 rows of x go past w in one launch. Where the tiles would need a packed copy of the longer operand (fp32, or
// rows that do not start on 16 bytes) up to 128 rows of the other stream it as it lies and join the slices of the contraction, unless the
// tiles, copies included, are estimated to be faster.
static bool streams(const LinearArgs& a, bool big_x) {
  const int64_t R = big_x ? a.M : a.N, S = big_x ? a.N : a.M;
  const bool dx = direct(a.dtype, a.x, a.ldx, a.K), dw = direct(a.dtype, a.w, a.ldw, a.K);
  if ((a.dtype != D_F32 && (big_x ? dx : dw)) || S > STREAM_SHORT || R < 4 * S || R < 256 || R > 1 << 29 || a.K < 256) return false;
  const double copied = (double)((dx ? 0 : a.M) + (dw ? 0 : a.N)) * a.K * (a.dtype == D_F32 ? 8 : 4);
  return stream_us(R, S, a.K, a.dtype) < product_us(a.M, a.N, a.K, 1, a.dtype, 0) + (copied > 0 ? 5.0 + copied / 4e6 : 0.0);
}

static int linear_stream(Ctx* ctx, hipStream_t st, const LinearArgs& a, bool big_x, void* ws, int64_t ws_bytes, int64_t* need) {
  Carve c(ws);
  const int64_t R = big_x ? a.M : a.N, S = big_x ? a.N : a.M;
  const void *big = big_x ? a.x : a.w, *small = big_x ? a.w : a.x;
  const int64_t ldb = big_x ? a.ldx : a.ldw, lds = big_x ? a.ldw : a.ldx;
  const int image = a.dtype == D_F32 ? D_PL3 : a.dtype;
  Mat img = image_of(c, image, S, a.K);
  int kchunk;
  const int slices = stream_slices(R, S, a.K, &kchunk);
  const int64_t n8 = round_up8(a.N);
  float* slabs = c.take<float>(slices * a.M * n8);
  *need = c.used;
  if (c.used > ws_bytes) return no_room(ctx, c.used);
  SCL_TRY(pack_image(ctx, st, a.dtype, image, small, lds, false, S, a.K, &img));
  SCL_TRY(stream_product(ctx, st, a.dtype, big, ldb, R, img, S, a.K, slabs, a.M * n8, big_x ? n8 : 1, big_x ? 1 : n8));
  Product p;
  p.M = a.M; p.N = a.N; p.K = a.K;
  p.out_type = p.res_type = a.dtype;
  p.bias = a.bias;
  p.act = a.act;
  if (a.res) { p.res = user_mat(a.res, a.ldr); p.beta = 1.f; }
  if (a.pre) p.pre = user_mat(a.pre, a.ldz);
  p.out = user_mat(a.y, a.ldy);
  p.slabs = slabs;
  return product_join(ctx, st, p, slices);
}

int linear_forward(Ctx* ctx, hipStream_t st, const LinearArgs& a, void* ws, int64_t ws_bytes, int64_t* need) {
  if (a.M > 0 && a.N > 0 && a.K > 0) {
    if (a.M <= 16) return linear_rows(ctx, st, a);
    const bool tiles_as_is = direct(a.dtype, a.x, a.ldx, a.K) && direct(a.dtype, a.w, a.ldw, a.K);
    if (!tiles_as_is && linear_is_small(a)) return linear_small(ctx, st, a);
    if (std::max(a.M, a.N) > MAX_ROWS) return ctx->fail(SCLENS_ERR_ARG, "linear: more than 2^30 - 64 rows");
    if (streams(a, false)) return linear_stream(ctx, st, a, false, ws, ws_bytes, need);
    if (streams(a, true)) return linear_stream(ctx, st, a, true, ws, ws_bytes, need);
  }
  Carve c(ws);
  if (a.K > MAX_CONTRACTION && a.M > 0 && a.N > 0) return ctx->fail(SCLENS_ERR_ARG, "linear: more than 2^25 columns");
  const bool planes = a.dtype == D_F32 && (a.K > MAX_CONTRACTION_F32 || planes_pay(a.M, a.N, a.K, (a.M + a.N) * a.K));
  const int image = planes ? D_PL3 : a.dtype;
  const bool dx = !planes && direct(a.dtype, a.x, a.ldx, a.K), dw = !planes && direct(a.dtype, a.w, a.ldw, a.K);
  Product p;
  p.type = image;
  p.out_type = p.res_type = a.dtype;
  p.M = a.M; p.N = a.N; p.K = a.K;
  p.A = dx ? user_mat(a.x, a.ldx) : image_of(c, image, a.M, a.K);
  p.B = dw ? user_mat(a.w, a.ldw) : image_of(c, image, a.N, a.K);
  p.slab_bytes = product_slab_bytes(a.M, a.N, a.K, 1, p.type, 0);
  if (p.slab_bytes) p.slabs = c.take<float>(p.slab_bytes / 4);
  *need = c.used;
  if (c.used > ws_bytes) return no_room(ctx, c.used);
  if (a.M == 0 || a.N == 0) return SCLENS_OK;
  SCL_TRY(pack_pair(ctx, st, a.dtype, image, a.x, a.ldx, a.M, dx ? nullptr : &p.A, a.w, a.ldw, a.N, dw ? nullptr : &p.B, a.K));
  p.bias = a.bias;
  p.act = a.act;
  if (a.res) { p.res = user_mat(a.res, a.ldr); p.beta = 1.f; }
  if (a.pre) p.pre = user_mat(a.pre, a.ldz);
  p.out = user_mat(a.y, a.ldy);
  return product(ctx, st, p);
}

// ------------------------------------------------------------------ linear, backward
// dz: 64 x 128 per workgroup, 8 columns per lane, its image (the same layout, padded with zeros to whole chunks) and the block's column
// sums in fp32, before dz is rounded. dz in 16 bits is one rounding of half a step per element, as the saved
// pre-activation and the gradient that comes in already are. Bound by HBM, two reads and a write per element: 8192 x 8192 bf16 77 us,
// 5.2 TB/s.
// fp16, whose steps are relative between 6e-5 and 65504 only, holds dz under a power of two that brings the largest |dy| to 2^14 .. 2^15 (no
// derivative exceeds 1.13): gradients of 1e-6 keep their eleven bits and those next to 65504 do not overflow. The products' epilogue takes
// it out again (`unscale`). k_largest finds it, a read of dy more; ReLU's dz is dy or zero and goes without.
constexpr int DZ_ROWS = 64, MAXIMA = 256;
__global__ __launch_bounds__(256) void k_largest(Mat dy, int64_t rows, int64_t cols, int tpr, unsigned* __restrict__ maxima) {
  __shared__ unsigned S[4];
  const int tid = threadIdx.x, tr = tid / tpr, tc = (tid % tpr) * 8, rpb = 256 / tpr;
  const int64_t step = (int64_t)gridDim.x * rpb;
  unsigned top = 0;  // finite fp16 magnitudes are ordered as their bits
  for (int64_t r = (int64_t)blockIdx.x * rpb + tr; r < rows; r += 4 * step)
    for (int64_t c = tc; c < cols; c += 8 * tpr) {
      const int n = (int)min((int64_t)8, cols - c);
      Raw8<D_F16> q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r + i * step < rows) q[i].load(dy, (r + i * step) * dy.ld + c, n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r + i * step >= rows) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned h = q[i].r[0][e] & 0x7fffu;
          if (h < 0x7c00u) top = max(top, h);
        }
      }
    }
  for (int w = 32; w > 0; w >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, w));
  if ((tid & 63) == 0) S[tid >> 6] = top;
  __syncthreads();
  if (tid == 0) maxima[blockIdx.x] = max(max(S[0], S[1]), max(S[2], S[3]));
}
template <int T>
__global__ __launch_bounds__(256) void k_dz(Mat dy, Mat z, int act, int64_t M, int64_t N, Mat img, float* __restrict__ part,
                                            const unsigned* __restrict__ maxima, int nmax, float* __restrict__ unscale) {
  __shared__ float L[16][132];
  __shared__ unsigned S[4];
  const int64_t nb = (N + 127) / 128, mb = blockIdx.x / nb;
  const int64_t m0 = mb * DZ_ROWS, n0 = (blockIdx.x % nb) * 128;
  const int tid = threadIdx.x, cc = (tid & 15) * 8, r0 = tid >> 4;
  const int64_t col = n0 + cc;
  const int nin = (int)max((int64_t)0, min((int64_t)8, N - col));
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.f;
  constexpr int NR = DZ_ROWS / 16;
  Raw8<T> g[NR], zz[NR];  // all loads first
  if (nin > 0) {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int64_t row = m0 + r0 + 16 * i;
      if (row < M) {
        g[i].load(dy, row * dy.ld + col, nin);
        if (act != ACT_NONE) zz[i].load(z, row * z.ld + col, nin);
      }
    }
  }
  float scale = 1.f;
  if constexpr (T == D_F16) {
    if (maxima) {
      unsigned top = tid < nmax ? maxima[tid] : 0;
      for (int w = 32; w > 0; w >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, w));
      if ((tid & 63) == 0) S[tid >> 6] = top;
      __syncthreads();
      top = max(max(S[0], S[1]), max(S[2], S[3]));
      const int k = top == 0 ? 0 : 14 - ilogbf(f16_to_f32((unsigned short)top));
      scale = ldexpf(1.f, k);
      if (blockIdx.x == 0 && tid == 0) *unscale = ldexpf(1.f, -k);
    }
  }
  if (nin > 0) {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int64_t row = m0 + r0 + 16 * i;
      if (row >= M) continue;
      float v[8];
      g[i].get(v);
      if (act != ACT_NONE) {
        float d[8];
        zz[i].get(d);
        act8<true>(d, act);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < nin ? v[e] * d[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += v[e];
      if constexpr (T == D_F16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= scale;
      }
      if (img.p) store8<T>(img, row * img.ld + col, 8, v);
    }
  }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) L[r0][cc + e] = sum[e];
  __syncthreads();
  if (tid < 128 && n0 + tid < N) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += L[r][tid];
    part[mb * N + n0 + tid] = s;
  }
}
// fp32 in planes, a 64 x 64 block: those of dz (contraction over the columns), those of its transpose (over the rows) and the column sums
__global__ __launch_bounds__(256) void k_dz_planes(Mat dy, Mat z, int act, int64_t M, int64_t N, Mat img, Mat imgT, float* __restrict__ part) {
  __shared__ float L[64][65];
  const int64_t nb = (N + 63) / 64, mb = blockIdx.x / nb;
  const int64_t m0 = mb * 64, n0 = (blockIdx.x % nb) * 64;
  const int tid = threadIdx.x, cc = (tid & 7) * 8;
  const int64_t col = n0 + cc;
  const int nin = (int)max((int64_t)0, min((int64_t)8, N - col));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int lr = i * 32 + (tid >> 3);
    const int64_t row = m0 + lr;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (row < M && nin > 0) {
      load8<D_F32>(dy, row * dy.ld + col, nin, v);
      if (act != ACT_NONE) {
        float zz[8];
        load8<D_F32>(z, row * z.ld + col, nin, zz);
        act8<true>(zz, act);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < nin) v[e] *= zz[e];
      }
    }
    if (img.p && row < M) store8<D_PL3>(img, row * img.ld + col, 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) L[lr][cc + e] = v[e];
  }
  __syncthreads();
  if (imgT.p) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int lc = i * 32 + (tid >> 3), lr = (tid & 7) * 8;
      if (n0 + lc < N) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = L[lr + e][lc];
        store8<D_PL3>(imgT, (n0 + lc) * imgT.ld + m0 + lr, 8, v);
      }
    }
  }
  if (part && tid < 64 && n0 + tid < N) {
    float s = 0.f;
    for (int r = 0; r < 64; ++r) s += L[r][tid];
    part[mb * N + n0 + tid] = s;
  }
}
template <int T>
__global__ __launch_bounds__(256) void k_colsum_join(const float* __restrict__ part, int64_t nmb, int64_t N, typename Elem<T>::type* __restrict__ out) {
  __shared__ double S[4][64];
  const int c = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + c;
  double s = 0.0;
  if (col < N)
#pragma unroll 8
    for (int64_t b = g; b < nmb; b += 4) s += (double)part[b * N + col];
  S[g][c] = s;
  __syncthreads();
  if (g == 0 && col < N) Elem<T>::st(out + col, (float)((S[0][c] + S[1][c]) + (S[2][c] + S[3][c])));
}

int linear_backward(Ctx* ctx, hipStream_t st, const LinearBwdArgs& a, void* ws, int64_t ws_bytes, int64_t* need) {
  if (a.M > 0 && a.N > 0 && backward_is_small(a)) return backward_small(ctx, st, a);
  if (a.N > (a.dtype == D_F32 && a.dx ? MAX_CONTRACTION_F32 : MAX_CONTRACTION) || a.K > MAX_CONTRACTION)
    return ctx->fail(SCLENS_ERR_ARG, "linear_backward: more than 2^25 columns (2^24 in an fp32 dx)");
  if (a.M > MAX_ROWS) return ctx->fail(SCLENS_ERR_ARG, "linear_backward: more than 2^30 - 64 rows");
  Carve c(ws);
  // fp32 in planes if each of the two products gains by it (dz, w and x are taken apart), whichever of them is asked for: a part of the gradients has
  // the bits that it has among all of them
  const bool planes = a.dtype == D_F32 && a.M <= MAX_CONTRACTION && planes_pay(a.M, a.K, a.N, a.M * a.N + a.N * a.K) &&
                      planes_pay(a.N, a.K, a.M, a.M * a.N + a.M * a.K);
  const int image = planes ? D_PL3 : a.dtype;
  const bool as_is = !planes && a.act == ACT_NONE && direct(a.dtype, a.dy, a.lddy, a.N);  // dz is dy
  const int rows_per = planes ? 64 : DZ_ROWS, cols_per = planes ? 64 : 128;
  const int64_t nmb = (a.M + rows_per - 1) / rows_per;
  // dz, w and x feed both products as they lie (w and x with their rows across the contraction), through a padded copy if they are not
  // on 16 bytes. Planes: the contraction contiguous, so dz both ways, w and x transposed.
  Mat dz, dzT, wT, xT;
  const bool w_as_is = !planes && direct(a.dtype, a.w, a.ldw, a.K), x_as_is = !planes && direct(a.dtype, a.x, a.ldx, a.K);
  if (a.dx || (a.dw && !planes)) dz = as_is ? user_mat(a.dy, a.lddy) : image_of(c, image, a.M, a.N);
  if (a.dx) wT = planes ? image_of(c, image, a.K, a.N) : (w_as_is ? user_mat(a.w, a.ldw) : image_of(c, image, a.N, a.K));
  if (a.dw && planes) dzT = image_of(c, image, a.N, a.M);
  if (a.dw) xT = planes ? image_of(c, image, a.K, a.M) : (x_as_is ? user_mat(a.x, a.ldx) : image_of(c, image, a.M, a.K));
  float* part = a.db ? c.take<float>(std::max<int64_t>(1, nmb * a.N)) : nullptr;
  const bool scaled = a.dtype == D_F16 && a.act > ACT_RELU && (a.dx || a.dw);
  unsigned* maxima = scaled ? c.take<unsigned>(MAXIMA) : nullptr;
  float* unscale = scaled ? c.take<float>(1) : nullptr;
  const int type = image;
  const int64_t slab_dx = a.dx ? product_slab_bytes(a.M, a.K, a.N, 1, type, 0) : 0;
  const int64_t slab_dw = a.dw ? product_slab_bytes(a.N, a.K, a.M, 1, type, 0) : 0;
  const int64_t slab = std::max(slab_dx, slab_dw);
  float* slabs = slab ? c.take<float>(slab / 4) : nullptr;
  *need = c.used;
  if (c.used > ws_bytes) return no_room(ctx, c.used);

  if (a.M > 0 && a.N > 0 && (a.db || (a.dw && planes) || ((a.dx || a.dw) && !as_is))) {
    const int64_t blocks = nmb * ((a.N + cols_per - 1) / cols_per);
    if (blocks >= 1 << 24) return ctx->fail(SCLENS_ERR_ARG, "linear_backward: too many elements");
    const Mat mdy = user_mat(a.dy, a.lddy), mz = user_mat(a.pre, a.ldz);
    Mat img = as_is ? Mat() : dz;
    const dim3 grid((unsigned)blocks), blk(256);
    int tpr = 1, nmax = 0;
    if (scaled) {
      while (tpr < 256 && 8 * tpr < a.N) tpr *= 2;
      nmax = (int)std::min<int64_t>(MAXIMA, std::max<int64_t>(1, a.M * tpr / 1024));
      SCL_RUN(ctx, k_largest, dim3((unsigned)nmax), blk, 0, st, mdy, a.M, a.N, tpr, maxima);
    }
    if (planes) SCL_RUN(ctx, k_dz_planes, grid, blk, 0, st, mdy, mz, a.act, a.M, a.N, img, dzT, part);
    else if (a.dtype == D_F32) SCL_RUN(ctx, k_dz<D_F32>, grid, blk, 0, st, mdy, mz, a.act, a.M, a.N, img, part, nullptr, 0, nullptr);
    else if (a.dtype == D_BF16) SCL_RUN(ctx, k_dz<D_BF16>, grid, blk, 0, st, mdy, mz, a.act, a.M, a.N, img, part, nullptr, 0, nullptr);
    else SCL_RUN(ctx, k_dz<D_F16>, grid, blk, 0, st, mdy, mz, a.act, a.M, a.N, img, part, maxima, nmax, unscale);
  }
  if (a.db && a.N > 0) {
    const dim3 grid((unsigned)((a.N + 63) / 64));
    if (a.dtype == D_F32) SCL_RUN(ctx, k_colsum_join<D_F32>, grid, dim3(256), 0, st, part, nmb, a.N, static_cast<float*>(a.db));
    else if (a.dtype == D_BF16) SCL_RUN(ctx, k_colsum_join<D_BF16>, grid, dim3(256), 0, st, part, nmb, a.N, static_cast<unsigned short*>(a.db));
    else SCL_RUN(ctx, k_colsum_join<D_F16>, grid, dim3(256), 0, st, part, nmb, a.N, static_cast<unsigned short*>(a.db));
  }
  if (!planes && a.K > 0) {
    const bool copy_w = a.dx && a.M > 0 && !w_as_is, copy_x = a.dw && a.N > 0 && !x_as_is;
    SCL_TRY(pack_pair(ctx, st, a.dtype, image, a.w, a.ldw, a.N, copy_w ? &wT : nullptr, a.x, a.ldx, a.M, copy_x ? &xT : nullptr, a.K));
  }
  Product p;
  p.type = type;
  p.out_type = p.res_type = a.dtype;
  p.slabs = slabs;
  p.slab_bytes = slab;
  p.scale = a.M > 0 && a.N > 0 ? unscale : nullptr;  // (an empty sum: nothing was scaled)
  if (a.dx && a.M > 0 && a.K > 0) {
    if (planes) SCL_TRY(pack_image(ctx, st, a.dtype, image, a.w, a.ldw, true, a.K, a.N, &wT));
    wT.across = !planes;
    p.M = a.M; p.N = a.K; p.K = a.N;
    p.A = dz; p.B = wT;
    p.out = user_mat(a.dx, a.lddx);
    SCL_TRY(product(ctx, st, p));
  }
  if (a.dw && a.N > 0 && a.K > 0) {
    if (planes) SCL_TRY(pack_image(ctx, st, a.dtype, image, a.x, a.ldx, true, a.K, a.M, &xT));
    xT.across = !planes;
    p.M = a.N; p.N = a.K; p.K = a.M;
    p.A = planes ? dzT : dz;
    p.A.across = !planes;
    p.B = xT;
    p.out = user_mat(a.dw, a.lddw);
    SCL_TRY(product(ctx, st, p));
  }
  return SCLENS_OK;
}

// ------------------------------------------------------------------ orthogonalize
// Both sides above 64 and one above 128: three products per step of the caller's layout, the two symmetric ones on the tiles on and below
// the diagonal. One 4096 x 4096 bf16 matrix, five steps: 8 + 18 us to scale it, 88 us per symmetric product (0.78 PFLOP/s of the lower
// half: 253 tiles of 192, one round), 136 us per full one (1.01 PFLOP/s). Four 1024 x 4096: A 36 us (144 tiles of 128 for 256 CUs), A A
// 14, the full one 45.
// |g|_F^2 of each matrix: partial sums in fp64 (fp32 squares of large entries overflow), added in a fixed order by whoever needs them.
// Bound by reading g: 8 columns per lane, tpr lanes to a row, four rows' loads on their way together (4096 x 4096 bf16: 8.2
// us, 24 with 2-byte loads).
template <int T>
__global__ __launch_bounds__(256) void k_sumsq(Mat src, int64_t rows, int64_t cols, int tpr, double* __restrict__ part) {
  __shared__ double S[256];
  const int tid = threadIdx.x, tr = tid / tpr, tc = (tid % tpr) * 8, rpb = 256 / tpr;
  const int64_t base = (int64_t)blockIdx.y * src.batch, step = (int64_t)gridDim.x * rpb;
  double s = 0.0;
  for (int64_t r = (int64_t)blockIdx.x * rpb + tr; r < rows; r += 4 * step)
    for (int64_t c = tc; c < cols; c += 8 * tpr) {
      const int n = (int)min((int64_t)8, cols - c);
      Raw8<T> q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r + i * step < rows) q[i].load(src, base + (r + i * step) * src.ld + c, n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r + i * step >= rows) continue;
        float v[8];
        q[i].get(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s += (double)v[e] * (double)v[e];
      }
    }
  S[tid] = s;
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if (tid < w) S[tid] += S[tid + w];
    __syncthreads();
  }
  if (tid == 0) part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = S[0];
}

// x0 = scale g / (|g|_F + eps), a 64 x 64 block: its image and the image of its transpose. `img` has the orientation of the source.
// Bound by one read and one write (4096 x 4096 bf16: 18 us, 3.7 TB/s).
template <int T, int IT>
__global__ __launch_bounds__(256) void k_orth_start(Mat src, int64_t rows, int64_t cols, const double* __restrict__ part, int nparts, double eps,
                                                    double scale, Mat img, Mat imgT) {
  __shared__ float L[64][65];
  __shared__ double S[4];
  const int64_t nb = (cols + 63) / 64, b = blockIdx.y;
  const int64_t m0 = (blockIdx.x / nb) * 64, n0 = (blockIdx.x % nb) * 64;
  const int tid = threadIdx.x, cc = (tid & 7) * 8;
  const int64_t col = n0 + cc;
  const int nin = (int)max((int64_t)0, min((int64_t)8, cols - col));
  Raw8<T> q[2];  // on their way while the norm is added up
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = m0 + i * 32 + (tid >> 3);
    if (row < rows && nin > 0) q[i].load(src, b * src.batch + row * src.ld + col, nin);
  }
  double s = 0.0;
  for (int i = tid; i < nparts; i += 256) s += part[b * nparts + i];
  for (int w = 32; w > 0; w >>= 1) s += __shfl_xor(s, w);
  if ((tid & 63) == 0) S[tid >> 6] = s;
  __syncthreads();
  const double f = scale / (sqrt((S[0] + S[1]) + (S[2] + S[3])) + eps);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int lr = i * 32 + (tid >> 3);
    const int64_t row = m0 + lr;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (row < rows && nin > 0) {
      q[i].get(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < nin ? (float)((double)v[e] * f) : 0.f;
    }
    if (row < rows) store8<IT>(img, b * img.batch + row * img.ld + col, 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) L[lr][cc + e] = v[e];
  }
  if (!imgT.p) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int lc = i * 32 + (tid >> 3), lr = (tid & 7) * 8;
    if (n0 + lc < cols) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = L[lr + e][lc];
      store8<IT>(imgT, b * imgT.batch + (n0 + lc) * imgT.ld + m0 + lr, 8, v);
    }
  }
}

// largest |a s + b s^3 + c s^5| over 0 <= s <= B: the singular values' bound after a step
double orth_step_bound(double a, double b, double c, double B) {
  auto f = [&](double s) { return std::fabs(((c * s * s + b) * s * s + a) * s); };
  double best = f(B);
  // a + 3 b q + 5 c q^2 = 0, q = s^2
  auto at = [&](double q) {
    if (q > 0 && q < B * B) best = std::max(best, f(std::sqrt(q)));
  };
  if (c != 0.0) {
    const double d = 9 * b * b - 20 * a * c;
    if (d >= 0) {
      at((-3 * b + std::sqrt(d)) / (10 * c));
      at((-3 * b - std::sqrt(d)) / (10 * c));
    }
  } else if (b != 0.0)
    at(-a / (3 * b));
  return best;
}

namespace {
// the power of two that brings a bound just under 2^14 (fp16 holds 65504: a factor of four is left for rounding)
double pow2_scale(double bound) { return std::ldexp(1.0, 13 - std::ilogb(std::max(bound, 1e-30))); }
}  // namespace

static int orth_chunk(Ctx* ctx, hipStream_t st, const OrthArgs& a, void* ws, int64_t ws_bytes, int64_t* need) {
  // x has m <= n: a matrix with more rows than columns is worked on transposed
  const bool tall = a.rows > a.cols;
  const int64_t m = tall ? a.cols : a.rows, n = tall ? a.rows : a.cols;
  // 16-bit inputs: x, A and b A + c A A between the products are fp16 under power-of-two scales from the bound of the singular values
  // (11 bits: eight times finer than bf16, so that what five steps amplify stays below the rounding of a bf16 result). fp32 inputs:
  // fp32, as it is or as three bf16 planes, exact.
  const bool wide = a.dtype == D_F32;
  const bool f32 = wide && n <= MAX_CONTRACTION &&  // planes
                   ((!tall && n > MAX_CONTRACTION_F32) || (planes_pay(m, n, m, 0, (int)a.batch) && planes_pay(m, m, n, 0, (int)a.batch, 1)));
  if (m > MAX_CONTRACTION_F32 || (!tall && n > MAX_CONTRACTION)) return ctx->fail(SCLENS_ERR_ARG, "orthogonalize: more than 2^25 columns");
  // The scales come from the bound, which may lie far above the singular values that are there. Those of a matrix of norm one reach 1 / sqrt(m);
  // `there` follows such a one through the steps, while it is small and at most to the bound. Held under the bound's scale, x is off by
  // (sqrt(m) + sqrt(n)) 2^-38 of the bound and P = b A + c A A by sqrt(m) 2^-36 of its bound (A's share included): up to the limits
  // here, and 8192 rows, less than 2^-11 of what is there.
  if (!wide) {
    double bound = 1.0, there = 1.0;  // (in units of 1 / sqrt(m))
    for (int t = 0; t < a.steps; ++t) {
      const double ca = std::fabs(a.coef[3 * t]), cb = std::fabs(a.coef[3 * t + 1]), cc = std::fabs(a.coef[3 * t + 2]);
      const double b2 = bound * bound, l = there * there / (double)m, grow = ca + (cb + cc * l) * l;
      if (bound > 0x1p14 * there || (cb + cc * b2) * b2 > 0x1p20 * grow)
        return ctx->fail(SCLENS_ERR_ARG, "orthogonalize: 16 bits between the products are too few for singular values that may grow this far; "
                                         "use fp32");
      bound = orth_step_bound(a.coef[3 * t], a.coef[3 * t + 1], a.coef[3 * t + 2], bound);
      there = std::min(there * grow, bound);
    }
  }
  const int IT = f32 ? D_PL3 : (wide ? D_F32 : D_F16), img_dtype = IT;
  Carve c(ws);
  const int64_t elems = m * n;
  const int nparts = (int)std::min<int64_t>(1024, std::max<int64_t>(1, elems / 8192));
  double* part = c.take<double>(a.batch * nparts);
  Mat X[2], XT[2];
  for (int i = 0; i < (a.steps > 1 ? 2 : 1); ++i) {
    // planes: x and its transpose, so that every product has the contraction contiguous; else x as it lies in memory
    X[i] = f32 ? image_of(c, img_dtype, m, n, a.batch) : image_of(c, img_dtype, a.rows, a.cols, a.batch);
    if (f32) XT[i] = image_of(c, img_dtype, n, m, a.batch);
  }
  Mat A = image_of(c, img_dtype, m, m, a.batch), P = image_of(c, img_dtype, m, m, a.batch);
  int64_t slab = std::max(product_slab_bytes(m, m, n, (int)a.batch, IT, 1), product_slab_bytes(m, m, m, (int)a.batch, IT, 1));
  slab = std::max(slab, f32 ? product_slab_bytes(m, n, m, (int)a.batch, IT, 0) : product_slab_bytes(a.rows, a.cols, m, (int)a.batch, IT, 0));
  float* slabs = slab ? c.take<float>(slab / 4) : nullptr;
  *need = c.used;
  if (c.used > ws_bytes) return no_room(ctx, c.used);

  const Mat src = user_mat(a.x, a.ldx, a.sx), dst = user_mat(a.y, a.ldy, a.sy);
  int tpr = 1;
  while (tpr < 256 && 8 * tpr < a.cols) tpr *= 2;
  const int64_t tiles = ((a.rows + 63) / 64) * ((a.cols + 63) / 64);
  if (tiles >= 1 << 24) return ctx->fail(SCLENS_ERR_ARG, "orthogonalize: too many elements");
  double bound = 1.0;
  double s_x = wide ? 1.0 : pow2_scale(bound);
  {
    const dim3 g1((unsigned)nparts, (unsigned)a.batch), g2((unsigned)tiles, (unsigned)a.batch), blk(256);
    const Mat i0 = tall && f32 ? XT[0] : X[0], i1 = tall && f32 ? X[0] : XT[0];
#define SCL_START(T, I)                                                                                                             \
  do {                                                                                                                              \
    SCL_RUN(ctx, k_sumsq<T>, g1, blk, 0, st, src, a.rows, a.cols, tpr, part);                                                       \
    SCL_RUN(ctx, k_orth_start<T, I>, g2, blk, 0, st, src, a.rows, a.cols, part, nparts, a.eps, s_x, i0, i1);                        \
  } while (0)
    if (f32) SCL_START(D_F32, D_PL3);
    else if (wide) SCL_START(D_F32, D_F32);
    else if (a.dtype == D_BF16) SCL_START(D_BF16, D_F16);
    else SCL_START(D_F16, D_F16);
#undef SCL_START
  }
  for (int t = 0; t < a.steps; ++t) {
    const double ca = a.coef[3 * t], cb = a.coef[3 * t + 1], cc = a.coef[3 * t + 2];
    const bool last = t + 1 == a.steps;
    const Mat &x = X[t & 1], &xt = XT[t & 1];
    const double next = orth_step_bound(ca, cb, cc, bound);
    const double s_a = wide ? 1.0 : pow2_scale(bound * bound);
    const double s_p = wide ? 1.0 : pow2_scale(std::fabs(cb) * bound * bound + std::fabs(cc) * bound * bound * bound * bound);
    const double s_n = wide || last ? 1.0 : pow2_scale(next);
    Product p;
    p.type = IT;
    p.batch = (int)a.batch;
    p.slabs = slabs;
    p.slab_bytes = slab;
    p.out_type = p.res_type = IT;
    p.symmetric = 1;
    p.M = p.N = m;
    // A = x x'
    p.K = n;
    p.A = p.B = x;
    p.A.across = p.B.across = tall && !f32;
    p.out = A;
    p.alpha = (float)(s_a / (s_x * s_x));
    SCL_TRY(product(ctx, st, p));
    // P = b A + c A A
    p.K = m;
    p.A = p.B = p.res = A;
    p.out = P;
    p.alpha = (float)(cc * s_p / (s_a * s_a));
    p.beta = (float)(cb * s_p / s_a);
    SCL_TRY(product(ctx, st, p));
    // x <- a x + P x (no planes, tall: the transpose of it, a x + x P, in the layout of the caller)
    p.symmetric = 0;
    p.res = x;
    p.alpha = (float)(s_n / (s_p * s_x));
    p.beta = (float)(ca * s_n / s_x);
    if (f32) {
      p.N = n;
      p.A = P;
      p.B = xt;
    } else {
      p.M = a.rows;
      p.N = a.cols;
      p.A = tall ? x : P;
      p.B = tall ? P : x;
      p.B.across = !tall;
    }
    if (last) {
      p.out_type = a.dtype;
      p.out = f32 && tall ? Mat() : dst;
      p.outT = f32 && tall ? dst : Mat();
    } else {
      p.out = X[(t + 1) & 1];
      p.outT = XT[(t + 1) & 1];
    }
    SCL_TRY(product(ctx, st, p));
    bound = next;
    s_x = s_n;
  }
  return SCLENS_OK;
}

int orthogonalize(Ctx* ctx, hipStream_t st, const OrthArgs& a, void* ws, int64_t ws_bytes, int64_t* need) {
  *need = 0;
  if (a.batch == 0 || a.rows == 0 || a.cols == 0) return SCLENS_OK;
  double bound = 1.0;
  for (int t = 0; t < a.steps; ++t) {
    bound = orth_step_bound(a.coef[3 * t], a.coef[3 * t + 1], a.coef[3 * t + 2], bound);
    // (fp32 holds its fourth power, the entries of A A)
    if (!(bound < 1e9)) return ctx->fail(SCLENS_ERR_ARG, "orthogonalize: these coefficients let the singular values grow without bound");
  }
  // 32768 matrices per launch (a grid holds 65535 in y). The last, shorter run may take another path than the others: what all of them
  // need is settled before the first one is launched.
  const int64_t chunk = 32768, size = a.dtype == D_F32 ? 4 : 2;
  for (int pass = a.batch > chunk ? 0 : 1; pass < 2; ++pass) {
    for (int64_t b0 = 0; b0 < a.batch; b0 += chunk) {
      OrthArgs b = a;
      b.batch = std::min(chunk, a.batch - b0);
      b.x = static_cast<const char*>(a.x) + b0 * a.sx * size;
      b.y = static_cast<char*>(a.y) + b0 * a.sy * size;
      const int64_t room = pass == 0 ? -1 : ws_bytes;  // -1: the size only
      int64_t n1 = 0;
      const int rc = orth_is_small(b) ? orth_small(ctx, st, b, ws, room, &n1) : orth_chunk(ctx, st, b, ws, room, &n1);
      *need = std::max(*need, n1);
      if (rc != SCLENS_OK && (pass == 1 || rc != SCLENS_ERR_WORKSPACE)) return rc;
    }
    if (*need > ws_bytes) return no_room(ctx, *need);
  }
  return SCLENS_OK;
}

}  // namespace scl
