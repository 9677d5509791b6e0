// Dense operators on device tensors: the product family behind sclens_hip_linear, sclens_hip_linear_backward and
// sclens_hip_orthogonalize (dense_gemm.hip: the products; dense_ops.hip: the operators).
#pragma once
#include "common.h"

namespace scl {

// A launch with its own status. (The runtime keeps one last error per thread: reading it after a launch would take, and report as this call's, one
// that the host framework has left there and not read yet.)
template <class T> struct Given { typedef T type; };
template <class... P>
int run_kernel(Ctx* ctx, void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t st, typename Given<P>::type... args) {
  void* at[] = {static_cast<void*>(&args)...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, at, lds, st);
  if (e != hipSuccess) (void)hipGetLastError();  // reported by this call's code
  SCL_HIP(ctx, e);
  return SCLENS_OK;
}
#define SCL_RUN(ctx, ...) SCL_TRY((run_kernel(ctx, __VA_ARGS__)))

// element types of the C ABI (SCLENS_DTYPE_*); D_PL3 is internal: an fp32 value held as three bf16 pieces in three planes
enum { D_F32 = 0, D_BF16 = 1, D_F16 = 2, D_PL3 = 3 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4 };

// A matrix on the device: element (r, c) of batch b at p + b * batch + r * ld + c; plane: distance of the planes of D_PL3.
struct Mat {
  void* p = nullptr;
  int64_t ld = 0, batch = 0, plane = 0;
  int vec = 0;  // 16-byte loads / stores of 8 columns are aligned
  int across = 0;  // an operand of a product whose rows run across the contraction: element (row r, column k) at k * ld + r; whole chunks
                   // of 8 rows have to exist
  int pad = 0;  // rows / columns up to the next multiple of 8 exist and are written as zeros (images of the library)
};

// C[b] = epilogue(alpha * A[b] B[b]'), A [M][K], B [N][K], the contraction contiguous or (Mat::across) the rows.
constexpr int64_t MAX_CONTRACTION = (int64_t)1 << 25;      // elements of an operand's row in the tiled products,
constexpr int64_t MAX_CONTRACTION_F32 = (int64_t)1 << 24;  // of an fp32 row along the contraction
constexpr int64_t MAX_ROWS = ((int64_t)1 << 30) - 64;      // rows: a grid's side holds fewer than 2^32 threads, 256 for 64 rows
struct Product {
  int type = D_BF16;  // of the operands; D_PL3: fp32 as three bf16 planes each, six products per term
  Mat A, B;
  int64_t M = 0, N = 0, K = 0;
  int batch = 1;
  int symmetric = 0;  // M == N and C is symmetric: tiles on / below the diagonal, mirrored
  // epilogue: v = alpha acc + bias[col]; pre = v; v = act(v) + beta res; out = v; outT (transposed) = v
  float alpha = 1.f, beta = 0.f;
  const float* scale = nullptr;  // device: alpha times this
  int act = ACT_NONE;
  const void* bias = nullptr;
  Mat res, pre, out, outT;
  int out_type = D_BF16, res_type = D_BF16;  // pre and bias have out_type
  // fp32 slabs of split contractions (see product_slab_bytes); nullptr: the contraction is never split
  float* slabs = nullptr;
  int64_t slab_bytes = 0;
};
int64_t product_slab_bytes(int64_t M, int64_t N, int64_t K, int batch, int type, int symmetric);
double product_us(int64_t M, int64_t N, int64_t K, int batch, int type, int symmetric);  // the plan's estimate
int product(Ctx* ctx, hipStream_t st, const Product& p);

// the join of slabs [slices][M][round_up8(N)] written by somebody else, through p's epilogue (p.slabs set; operands only for fp32 NaN)
int product_join(Ctx* ctx, hipStream_t st, const Product& p, int slices);

// dense_stream.hip: products with one short side (linear_forward has the rule)
constexpr int64_t STREAM_SHORT = 128;
int stream_slices(int64_t R, int64_t S, int64_t K, int* kchunk);
double stream_us(int64_t R, int64_t S, int64_t K, int dtype);
int stream_product(Ctx* ctx, hipStream_t st, int dtype, const void* big, int64_t ldb, int64_t R, const Mat& small, int64_t S, int64_t K,
                   float* slabs, int64_t slab, int64_t sr, int64_t ss);

// Image of src (element (r, k) at r * ld + k, transposed: k * ld + r), rows x K, K padded with zeros to image_ld(K): of its own type, or
// (D_PL3, from fp32) three bf16 planes
static inline int64_t image_ld(int64_t K) { return round_up(K > 0 ? K : 1, 64); }
static inline int64_t image_elems(int64_t rows, int64_t K) { return round_up(rows, 8) * image_ld(K); }
int pack_image(Ctx* ctx, hipStream_t st, int dtype, int image, const void* src, int64_t ld, bool transposed, int64_t rows, int64_t K, Mat* img);
// two of equal K, not transposed, in one launch; an image that is nullptr is left out
int pack_pair(Ctx* ctx, hipStream_t st, int dtype, int image, const void* a, int64_t lda, int64_t rows_a, Mat* img_a, const void* b, int64_t ldb,
              int64_t rows_b, Mat* img_b, int64_t K);

struct LinearArgs {
  int dtype = D_F32, act = ACT_NONE;
  int64_t M = 0, N = 0, K = 0;
  const void *x = nullptr, *w = nullptr, *bias = nullptr, *res = nullptr;
  void *y = nullptr, *pre = nullptr;
  int64_t ldx = 0, ldw = 0, ldr = 0, ldy = 0, ldz = 0;
};
struct LinearBwdArgs {
  int dtype = D_F32, act = ACT_NONE;
  int64_t M = 0, N = 0, K = 0;
  const void *dy = nullptr, *x = nullptr, *w = nullptr, *pre = nullptr;
  void *dx = nullptr, *dw = nullptr, *db = nullptr;
  int64_t lddy = 0, ldx = 0, ldw = 0, ldz = 0, lddx = 0, lddw = 0;
};
struct OrthArgs {
  int dtype = D_F32;
  int64_t batch = 0, rows = 0, cols = 0;
  const void* x = nullptr;
  void* y = nullptr;
  int64_t sx = 0, ldx = 0, sy = 0, ldy = 0;
  int steps = 0;
  const double* coef = nullptr;  // steps x (a, b, c), host
  double eps = 0;
};
double orth_step_bound(double a, double b, double c, double B);  // the singular values' bound after a step
bool orth_is_small(const OrthArgs& a);  // dense_orth.hip: both sides at most 128 (and few steps), or a short side of at most 64
int orth_small(Ctx* ctx, hipStream_t st, const OrthArgs& a, void* ws, int64_t ws_bytes, int64_t* need);
int linear_rows(Ctx* ctx, hipStream_t st, const LinearArgs& a);  // M <= 16

bool linear_is_small(const LinearArgs& a);  // dense_small.hip: one launch, any address, no scratch
bool backward_is_small(const LinearBwdArgs& a);
int linear_small(Ctx* ctx, hipStream_t st, const LinearArgs& a);
int backward_small(Ctx* ctx, hipStream_t st, const LinearBwdArgs& a);

// *need: bytes of scratch the call wants; launched only if ws_bytes >= *need (SCLENS_ERR_WORKSPACE otherwise)
int linear_forward(Ctx* ctx, hipStream_t st, const LinearArgs& a, void* ws, int64_t ws_bytes, int64_t* need);
int linear_backward(Ctx* ctx, hipStream_t st, const LinearBwdArgs& a, void* ws, int64_t ws_bytes, int64_t* need);
int orthogonalize(Ctx* ctx, hipStream_t st, const OrthArgs& a, void* ws, int64_t ws_bytes, int64_t* need);

// scratch handed out in order, 256-byte aligned; with base == nullptr only the sizes are summed
struct Carve {
  char* base;
  int64_t used = 0;
  explicit Carve(void* b) : base(static_cast<char*>(b)) {}
  template <class T>
  T* take(int64_t count) {
    const int64_t off = used;
    used += round_up(count * (int64_t)sizeof(T), 256);
    return base ? reinterpret_cast<T*>(base + off) : nullptr;
  }
};

}  // namespace scl
