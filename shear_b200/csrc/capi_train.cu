// C ABI of the operators that train a table of vectors (lookup, FP8 product,
// distillation): argument checks before any launch.  These calls enqueue and
// return; see the header on how device-side errors are reported.
#include <cstdarg>
#include <cstdio>

#include "kernels.h"

using namespace tessa;

namespace {

int bad(int code, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_last_error(code, buf);
}

#define TRY(expr)                \
  do {                           \
    int _r = (expr);             \
    if (_r != TESSA_OK) return _r; \
  } while (0)

typedef unsigned long long ull;

uint32_t elem_bytes(uint32_t dtype) { return dtype == TESSA_F32 ? 4u : 2u; }

int check_dtype(const char* what, uint32_t dtype) {
  if (dtype > TESSA_F16) return bad(TESSA_ERR_INVALID_ARG, "%s: unknown element type %u", what, dtype);
  return TESSA_OK;
}

// A matrix argument: pointer present and element-aligned, stride of at least a row.
int check_matrix(const char* what, const void* p, uint64_t rows, uint64_t cols, uint64_t stride, uint32_t dtype) {
  TRY(check_dtype(what, dtype));
  if (rows == 0 || cols == 0) return TESSA_OK;
  if (!p) return bad(TESSA_ERR_INVALID_ARG, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(p) % elem_bytes(dtype))
    return bad(TESSA_ERR_INVALID_ARG, "%s: not aligned to its element type", what);
  if (rows > 1 && stride < cols)
    return bad(TESSA_ERR_INVALID_ARG, "%s: stride %llu below %llu columns", what, (ull)stride, (ull)cols);
  if (stride > (1ull << 40)) return bad(TESSA_ERR_UNSUPPORTED, "%s: stride %llu above 2^40", what, (ull)stride);
  return TESSA_OK;
}

int check_ids(const void* ids, uint32_t id_bits, uint64_t count) {
  if (id_bits != 32 && id_bits != 64) return bad(TESSA_ERR_INVALID_ARG, "ids of %u bits: 32 or 64", id_bits);
  if (count && !ids) return bad(TESSA_ERR_INVALID_ARG, "ids: null pointer");
  if (reinterpret_cast<uintptr_t>(ids) % (id_bits / 8))
    return bad(TESSA_ERR_INVALID_ARG, "ids: not aligned to their type");
  return TESSA_OK;
}

int check_workspace(const void* ws, uint64_t have, uint64_t need) {
  if (need == 0) return TESSA_OK;
  if (!ws || have < need)
    return bad(TESSA_ERR_INVALID_ARG, "workspace of %llu bytes, %llu needed", (ull)(ws ? have : 0), (ull)need);
  if (reinterpret_cast<uintptr_t>(ws) % 256) return bad(TESSA_ERR_INVALID_ARG, "workspace not 256-byte aligned");
  return TESSA_OK;
}

// Whether any row at p (`bytes` long, p_step from one to the next) shares memory
// with a row at q, other than being all of the same row.
bool rows_overlap(const void* p, uint64_t p_step, const void* q, uint64_t q_step, uint64_t rows, uint64_t bytes) {
  if (rows == 0 || bytes == 0) return false;
  const uint64_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q), last = rows - 1;
  if (a + last * p_step + bytes <= b || b + last * q_step + bytes <= a) return false;
  if (a == b && (rows == 1 || p_step == q_step)) return false;
  if (rows == 1) return true;
  if (p_step == q_step) {  // side by side in one wider matrix, or not
    const uint64_t d = (a < b ? b - a : a - b) % p_step;
    return d < bytes || p_step - d < bytes;
  }
  for (uint64_t i = 0, j = 0; i < rows && j < rows;) {
    const uint64_t x = a + i * p_step, y = b + j * q_step;
    if (x + bytes <= y) ++i;
    else if (y + bytes <= x) ++j;
    else return true;
  }
  return false;
}

int launched(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return TESSA_OK;
  return bad(e == cudaErrorMemoryAllocation ? TESSA_ERR_OOM : TESSA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

constexpr uint64_t kMaxIds = 1ull << 31;          // sorted positions are 32-bit
constexpr uint64_t kMaxMatrix = (1ull << 31) - 1;  // TMA coordinates and tile counts are 32-bit
constexpr uint64_t kMaxTableRows = 0xfffffffeull;  // one key above the last row marks padding
constexpr uint32_t kMaxDim = 0xfffffc00u;          // columns are counted in 32 bits, by steps of up to 256

int check_dim(uint32_t dim) {
  if (dim > kMaxDim) return bad(TESSA_ERR_UNSUPPORTED, "rows of %u columns: at most 2^32 - 1024", dim);
  return TESSA_OK;
}

}  // namespace

extern "C" {

int tessa_embedding_lookup(tessa_ctx* ctx, const tessa_lookup_args* args, void* stream) {
  if (!ctx || !args) return bad(TESSA_ERR_INVALID_ARG, "null argument");
  const tessa_lookup_args& a = *args;
  TRY(check_matrix("table", a.table, a.table_rows, a.dim, a.table_stride, a.dtype));
  TRY(check_matrix("out", a.out, a.count, a.dim, a.out_stride, a.out_dtype));
  TRY(check_ids(a.ids, a.id_bits, a.count));
  TRY(check_dim(a.dim));
  if (a.table_rows > kMaxTableRows) return bad(TESSA_ERR_UNSUPPORTED, "table of %llu rows", (ull)a.table_rows);
  if (a.count >= kMaxIds) return bad(TESSA_ERR_UNSUPPORTED, "%llu ids: below 2^31 are supported", (ull)a.count);
  AsyncCtx c;
  TRY(async_begin(ctx, &c));
  if (a.count == 0 || a.dim == 0) return TESSA_OK;
  return launched("embedding lookup", launch_embedding_lookup(a, c, (cudaStream_t)stream));
}

int tessa_embedding_grad_workspace(uint64_t count, uint64_t table_rows, uint32_t dim, uint64_t* bytes) {
  if (!bytes) return bad(TESSA_ERR_INVALID_ARG, "null argument");
  TRY(check_dim(dim));
  *bytes = embedding_grad_workspace(count, table_rows, dim);
  return TESSA_OK;
}

int tessa_embedding_grad(tessa_ctx* ctx, const tessa_lookup_grad_args* args, void* workspace,
                         uint64_t workspace_bytes, void* stream) {
  if (!ctx || !args) return bad(TESSA_ERR_INVALID_ARG, "null argument");
  const tessa_lookup_grad_args& a = *args;
  TRY(check_matrix("dout", a.dout, a.count, a.dim, a.dout_stride, a.dtype));
  TRY(check_matrix("grad", a.grad, a.table_rows, a.dim, a.grad_stride, a.grad_dtype));
  TRY(check_ids(a.ids, a.id_bits, a.count));
  TRY(check_dim(a.dim));
  if (a.accumulate > 1) return bad(TESSA_ERR_INVALID_ARG, "accumulate %u: 0 or 1", a.accumulate);
  if (a.table_rows > kMaxTableRows) return bad(TESSA_ERR_UNSUPPORTED, "table of %llu rows", (ull)a.table_rows);
  if (a.count >= kMaxIds) return bad(TESSA_ERR_UNSUPPORTED, "%llu ids: below 2^31 are supported", (ull)a.count);
  TRY(check_workspace(workspace, workspace_bytes, embedding_grad_workspace(a.count, a.table_rows, a.dim)));
  AsyncCtx c;
  TRY(async_begin(ctx, &c));
  if (a.table_rows == 0 || a.dim == 0) return TESSA_OK;
  return launched("embedding gradient", launch_embedding_grad(a, workspace, c, (cudaStream_t)stream));
}

int tessa_quantize_fp8(tessa_ctx* ctx, const tessa_fp8_quantize_args* args, void* stream) {
  if (!ctx || !args) return bad(TESSA_ERR_INVALID_ARG, "null argument");
  const tessa_fp8_quantize_args& a = *args;
  TRY(check_matrix("x", a.x, a.rows, a.cols, a.stride, a.dtype));
  if (a.rows > kMaxMatrix || a.cols > kMaxMatrix)
    return bad(TESSA_ERR_UNSUPPORTED, "matrix of %llu x %llu: both below 2^31", (ull)a.rows, (ull)a.cols);
  if (a.rows * ((a.cols + 127) / 128) > kMaxMatrix)
    return bad(TESSA_ERR_UNSUPPORTED, "matrix of %llu x %llu is too large", (ull)a.rows, (ull)a.cols);
  if (!a.codes != !a.scales || !a.codes_t != !a.scales_t || (!a.codes && !a.codes_t)) {
    if (a.rows && a.cols) return bad(TESSA_ERR_INVALID_ARG, "codes and scales come in pairs, one pair at least");
  }
  if (reinterpret_cast<uintptr_t>(a.codes) % 16 || reinterpret_cast<uintptr_t>(a.codes_t) % 16)
    return bad(TESSA_ERR_INVALID_ARG, "codes must start on a 16-byte boundary");
  AsyncCtx c;
  TRY(async_begin(ctx, &c));
  if (a.rows == 0 || a.cols == 0) return TESSA_OK;
  return launched("FP8 quantizer", launch_quantize_fp8(a, c, (cudaStream_t)stream));
}

int tessa_matmul_fp8_workspace(tessa_ctx* ctx, uint64_t m, uint64_t n, uint64_t k, uint64_t* bytes) {
  if (!ctx || !bytes) return bad(TESSA_ERR_INVALID_ARG, "null argument");
  if (m > kMaxMatrix || n > kMaxMatrix || k > kMaxMatrix)
    return bad(TESSA_ERR_UNSUPPORTED, "product of %llu x %llu x %llu: each below 2^31", (ull)m, (ull)n, (ull)k);
  *bytes = fp8_matmul_workspace(m, n, k, ctx_sm_count(ctx));
  return TESSA_OK;
}

int tessa_matmul_fp8(tessa_ctx* ctx, const tessa_fp8_matmul_args* args, void* workspace, uint64_t workspace_bytes,
                     void* stream) {
  if (!ctx || !args) return bad(TESSA_ERR_INVALID_ARG, "null argument");
  const tessa_fp8_matmul_args& a = *args;
  TRY(check_matrix("out", a.out, a.m, a.n, a.out_stride, a.out_dtype));
  uint64_t need = 0;
  TRY(tessa_matmul_fp8_workspace(ctx, a.m, a.n, a.k, &need));
  if (a.k % 16) return bad(TESSA_ERR_INVALID_ARG, "k=%llu: rows of codes are a multiple of 16", (ull)a.k);
  if (fp8_matmul_units(a.m, a.n, a.k, ctx_sm_count(ctx)) > kMaxMatrix)
    return bad(TESSA_ERR_UNSUPPORTED, "product of %llu x %llu is too large", (ull)a.m, (ull)a.n);
  if (a.m && a.n && a.k) {
    if (!a.a_codes || !a.a_scales || !a.b_codes || !a.b_scales) return bad(TESSA_ERR_INVALID_ARG, "null codes or scales");
    if (reinterpret_cast<uintptr_t>(a.a_codes) % 16 || reinterpret_cast<uintptr_t>(a.b_codes) % 16)
      return bad(TESSA_ERR_INVALID_ARG, "codes must start on a 16-byte boundary");
    if (reinterpret_cast<uintptr_t>(a.a_scales) % 4 || reinterpret_cast<uintptr_t>(a.b_scales) % 4)
      return bad(TESSA_ERR_INVALID_ARG, "scales must start on a 4-byte boundary");
  }
  TRY(check_workspace(workspace, workspace_bytes, need));
  AsyncCtx c;
  TRY(async_begin(ctx, &c));
  if (a.m == 0 || a.n == 0) return TESSA_OK;
  return launched("FP8 product", launch_matmul_fp8(a, workspace, c, (cudaStream_t)stream));
}

int tessa_distill_topk_workspace(const tessa_distill_args* args, uint64_t* bytes) {
  if (!args || !bytes) return bad(TESSA_ERR_INVALID_ARG, "null argument");
  TRY(check_dtype("logits", args->dtype));
  *bytes = distill_workspace(args->rows, args->vocab, args->dtype, args->k, args->grad != nullptr);
  return TESSA_OK;
}

int tessa_distill_topk(tessa_ctx* ctx, const tessa_distill_args* args, void* workspace, uint64_t workspace_bytes,
                       void* stream) {
  if (!ctx || !args) return bad(TESSA_ERR_INVALID_ARG, "null argument");
  const tessa_distill_args& a = *args;
  TRY(check_matrix("logits", a.logits, a.rows, a.vocab, a.stride, a.dtype));
  if (a.grad) TRY(check_matrix("grad", a.grad, a.rows, a.vocab, a.grad_stride, a.dtype));
  if (a.grad == a.logits && a.rows > 1 && a.grad_stride != a.stride)
    return bad(TESSA_ERR_INVALID_ARG, "a gradient in place of the logits needs their stride");
  const uint64_t bytes = elem_bytes(a.dtype);
  if (a.grad && rows_overlap(a.logits, a.stride * bytes, a.grad, a.grad_stride * bytes, a.rows, a.vocab * bytes))
    return bad(TESSA_ERR_INVALID_ARG, "the gradient overlaps the logits: it may be in their place, or apart");
  if (a.k > TESSA_MAX_DISTILL_K) return bad(TESSA_ERR_INVALID_ARG, "list of %u entries: at most %d", a.k, TESSA_MAX_DISTILL_K);
  if (a.vocab > kMaxTableRows) return bad(TESSA_ERR_UNSUPPORTED, "%llu logits a row", (ull)a.vocab);
  if (a.rows > (1ull << 27)) return bad(TESSA_ERR_UNSUPPORTED, "%llu rows: at most 2^27", (ull)a.rows);
  TRY(check_ids(a.teacher_ids, a.id_bits, a.rows * a.k));
  if (a.rows * a.k && !a.teacher_logits) return bad(TESSA_ERR_INVALID_ARG, "teacher logits: null pointer");
  if (!(a.temperature > 0.0f) || a.temperature > 3.0e38f)
    return bad(TESSA_ERR_INVALID_ARG, "temperature %g: a positive number", (double)a.temperature);
  if (1.44269504f / a.temperature > 3.402823466e38f)  // log2(e) / tau is a factor: infinite, it makes 0 * inf of equal logits
    return bad(TESSA_ERR_INVALID_ARG, "temperature %g: at least 4.24e-39", (double)a.temperature);
  TRY(check_workspace(workspace, workspace_bytes, distill_workspace(a.rows, a.vocab, a.dtype, a.k, a.grad != nullptr)));
  AsyncCtx c;
  TRY(async_begin(ctx, &c));
  if (a.rows == 0) return TESSA_OK;
  return launched("distillation", launch_distill(a, workspace, c, (cudaStream_t)stream));
}

}  // extern "C"
