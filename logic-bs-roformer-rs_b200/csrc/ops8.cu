// C entry points of the 8-bit operators: argument checks before any device
// work, then one kernel launch each.
#include <string>

#include "../../include/lbrr_gpu.h"
#include "kernels.h"

using namespace lbrr;

namespace {

int bad(const char* op, const std::string& what) {
  return lbrr_set_error_for_host(LBRR_ERR_INVALID, (std::string(op) + ": " + what).c_str());
}
int launched(const char* op, cudaError_t e) {
  if (e == cudaSuccess) return LBRR_OK;
  cudaGetLastError();  // reported here: the next call's launch does not find it
  return lbrr_set_error_for_host(LBRR_ERR_CUDA, (std::string(op) + ": " + cudaGetErrorString(e)).c_str());
}

constexpr int64_t kMaxRows = 1ll << 30;
constexpr int64_t kMaxCols = 65535ll * 128;  // a grid dimension's worth of 128-column blocks
constexpr int64_t kMaxLd = 1ll << 36;  // elements between rows

bool known_type(int32_t t) { return t == LBRR_DT_F32 || t == LBRR_DT_F16 || t == LBRR_DT_BF16; }
size_t size_of(int32_t t) { return t == LBRR_DT_F32 ? 4 : 2; }
int64_t blocks(int64_t n) { return (n + 127) / 128; }
// A matrix whose rows start ld elements apart, of a type of `size` bytes.
bool ok_matrix(const void* p, int64_t ld, int64_t cols, size_t size) {
  return p && ld >= cols && ld <= kMaxLd && reinterpret_cast<uintptr_t>(p) % size == 0;
}
bool ok_operand8(const void* p, int64_t ld, int64_t cols) {
  return ok_matrix(p, ld, cols, 1) && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 16 == 0;
}

// Checks shared by the two products.
int check_product(const char* op, const uint8_t* a, int64_t lda, const float* a_scales, int64_t ldas,
                  const uint8_t* w, int64_t ldw, const float* w_scales, int64_t ldws, const float* bias, int64_t m,
                  int64_t n, int64_t k) {
  if (!ok_operand8(a, lda, k) || !ok_operand8(w, ldw, k))
    return bad(op, "8-bit operands need rows that start on 16-byte boundaries, at least k bytes apart");
  if (!ok_matrix(a_scales, ldas, m, 4)) return bad(op, "bad a_scales");
  if (!ok_matrix(w_scales, ldws, blocks(n), 4)) return bad(op, "bad w_scales");
  if (reinterpret_cast<uintptr_t>(bias) % 4 != 0) return bad(op, "misaligned bias");
  if (blocks(m) * blocks(n) > (1ll << 30)) return bad(op, "more than 2^30 tiles of 128 x 128");
  return LBRR_OK;
}

// The per-device status word of the products.  Its first use on a device
// allocates, which a stream capture does not allow.
int status_word(const char* op, cudaStream_t st, int** status) {
  *status = op_status(true);
  if (!*status) {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(st, &cs) != cudaSuccess || cs != cudaStreamCaptureStatusNone) {
      cudaGetLastError();  // the default stream beside a blocking one's capture cannot be asked
      return lbrr_set_error_for_host(
          LBRR_ERR_STATE,
          (std::string(op) + ": call a per-op entry point once on this device before recording it into a graph")
              .c_str());
    }
    *status = op_status();
  }
  if (!*status) return lbrr_set_error_for_host(LBRR_ERR_CUDA, "op status allocation failed");
  return LBRR_OK;
}

}  // namespace

extern "C" int lbrr_op_quant8(const void* x, int32_t x_type, int64_t ldx, int64_t rows, int64_t cols,
                              int32_t block_rows, uint8_t* q, int64_t ldq, float* scales, int64_t lds, void* stream) {
  const char* op = "lbrr_op_quant8";
  if (!known_type(x_type)) return bad(op, "unknown x_type");
  if (block_rows != 1 && block_rows != 128) return bad(op, "block_rows must be 1 or 128");
  if (rows < 0 || rows > kMaxRows || cols <= 0 || cols > kMaxCols) return bad(op, "bad rows or cols");
  if (rows == 0) return LBRR_OK;
  if (block_rows == 128 && blocks(rows) * blocks(cols) > (1ll << 30)) return bad(op, "more than 2^30 blocks");
  if (!ok_matrix(x, ldx, cols, size_of(x_type))) return bad(op, "bad x");
  if (!ok_matrix(q, ldq, cols, 1)) return bad(op, "bad q");
  if (!ok_matrix(scales, lds, block_rows == 1 ? rows : blocks(rows), 4)) return bad(op, "bad scales");
  return launched(op, quant8(x, static_cast<Elem>(x_type), ldx, static_cast<int>(rows), static_cast<int>(cols),
                             block_rows, q, ldq, scales, lds, static_cast<cudaStream_t>(stream)));
}

extern "C" int lbrr_op_add_norm_quant8(const void* x, int32_t x_type, int64_t ldx, const void* resid,
                                       int32_t resid_type, int64_t ldr, const float* gamma, float eps, void* y,
                                       int64_t ldy, uint8_t* q, int64_t ldq, float* scales, int64_t lds, int64_t rows,
                                       int64_t cols, void* stream) {
  const char* op = "lbrr_op_add_norm_quant8";
  if (!known_type(x_type) || !known_type(resid_type)) return bad(op, "unknown x_type or resid_type");
  if (resid_type != x_type && resid_type != LBRR_DT_F32) return bad(op, "resid_type must be x_type or LBRR_DT_F32");
  if (rows < 0 || rows > kMaxRows || cols <= 0 || cols > kNorm8MaxCols)
    return bad(op, "bad rows, or cols outside 1.." + std::to_string(kNorm8MaxCols));
  if (!(eps >= 0.0f) || eps > 1.0f) return bad(op, "eps must be in [0, 1]");
  if (y && !resid) return bad(op, "y (the sum) needs resid");
  if (rows == 0) return LBRR_OK;
  if (!ok_matrix(x, ldx, cols, size_of(x_type))) return bad(op, "bad x");
  if (resid && !ok_matrix(resid, ldr, cols, size_of(resid_type))) return bad(op, "bad resid");
  if (y && !ok_matrix(y, ldy, cols, size_of(resid_type))) return bad(op, "bad y");
  if (!gamma || reinterpret_cast<uintptr_t>(gamma) % 4 != 0) return bad(op, "bad gamma");
  if (!ok_matrix(q, ldq, cols, 1)) return bad(op, "bad q");
  if (!ok_matrix(scales, lds, rows, 4)) return bad(op, "bad scales");
  if (y && ((y == resid && rows > 1 && ldy != ldr) || (y == x && (resid_type != x_type || (rows > 1 && ldy != ldx)))))
    return bad(op, "y in place needs the input's type and distance between rows");
  AddNorm8 a{};
  a.x = x;
  a.x_type = static_cast<Elem>(x_type);
  a.ldx = ldx;
  a.resid = resid;
  a.resid_type = static_cast<Elem>(resid_type);
  a.ldr = ldr;
  a.gamma = gamma;
  a.eps = eps;
  a.y = y;
  a.ldy = ldy;
  a.q = q;
  a.ldq = ldq;
  a.scales = scales;
  a.lds = lds;
  a.rows = static_cast<int>(rows);
  a.cols = static_cast<int>(cols);
  return launched(op, add_norm_quant8(a, static_cast<cudaStream_t>(stream)));
}

static Gemm8 product(const uint8_t* a, int64_t lda, const float* a_scales, int64_t ldas, const uint8_t* w,
                     int64_t ldw, const float* w_scales, int64_t ldws, const float* bias, int64_t m, int64_t n,
                     int64_t k) {
  Gemm8 g{};
  g.a = a;
  g.lda = lda;
  g.a_scales = a_scales;
  g.ldas = ldas;
  g.w = w;
  g.ldw = ldw;
  g.w_scales = w_scales;
  g.ldws = ldws;
  g.bias = bias;
  g.m = static_cast<int>(m);
  g.n = static_cast<int>(n);
  g.k = static_cast<int>(k);
  return g;
}

extern "C" int lbrr_op_gemm8(const uint8_t* a, int64_t lda, const float* a_scales, int64_t ldas, const uint8_t* w,
                             int64_t ldw, const float* w_scales, int64_t ldws, const float* bias, const void* resid,
                             int64_t ldr, void* out, int32_t out_type, int64_t ldo, int64_t m, int64_t n, int64_t k,
                             void* stream) {
  const char* op = "lbrr_op_gemm8";
  if (!known_type(out_type)) return bad(op, "unknown out_type");
  if (m < 0 || m > kMaxRows || n <= 0 || n > kMaxCols || k <= 0 || k > kMaxCols) return bad(op, "bad m, n or k");
  if (m == 0) return LBRR_OK;
  if (int rc = check_product(op, a, lda, a_scales, ldas, w, ldw, w_scales, ldws, bias, m, n, k)) return rc;
  if (!ok_matrix(out, ldo, n, size_of(out_type))) return bad(op, "bad out");
  if (resid && !ok_matrix(resid, ldr, n, size_of(out_type))) return bad(op, "bad resid");
  if (resid == out && m > 1 && ldr != ldo) return bad(op, "out in place needs resid's distance between rows");
  Gemm8 g = product(a, lda, a_scales, ldas, w, ldw, w_scales, ldws, bias, m, n, k);
  g.resid = resid;
  g.ldr = ldr;
  g.out = out;
  g.out_type = static_cast<Elem>(out_type);
  g.ldo = ldo;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int* status = nullptr;
  if (int rc = status_word(op, st, &status)) return rc;
  return launched(op, gemm8(g, status, st));
}

extern "C" int lbrr_op_gemm8_gelu_quant8(const uint8_t* a, int64_t lda, const float* a_scales, int64_t ldas,
                                         const uint8_t* w, int64_t ldw, const float* w_scales, int64_t ldws,
                                         const float* bias, uint8_t* q, int64_t ldq, float* scales, int64_t lds,
                                         int64_t m, int64_t n, int64_t k, void* stream) {
  const char* op = "lbrr_op_gemm8_gelu_quant8";
  if (m < 0 || m > kMaxRows || n <= 0 || n > kMaxCols || k <= 0 || k > kMaxCols) return bad(op, "bad m, n or k");
  if (m == 0) return LBRR_OK;
  if (int rc = check_product(op, a, lda, a_scales, ldas, w, ldw, w_scales, ldws, bias, m, n, k)) return rc;
  if (!ok_matrix(q, ldq, n, 1)) return bad(op, "bad q");
  if (!ok_matrix(scales, lds, m, 4)) return bad(op, "bad scales");
  Gemm8 g = product(a, lda, a_scales, ldas, w, ldw, w_scales, ldws, bias, m, n, k);
  g.q = q;
  g.ldq = ldq;
  g.scales = scales;
  g.lds = lds;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int* status = nullptr;
  if (int rc = status_word(op, st, &status)) return rc;
  return launched(op, gemm8(g, status, st));
}
