// C ABI of llmopt_float8.h: checks, the choice of kernels, and launches.
#include <stdarg.h>
#include <stdio.h>

#include "../../../include/llmopt_float8.h"
#include "../../../include/llmopt_qlinear.h"
#include "f8_common.hpp"

namespace {

using namespace llmopt;

thread_local char g_error[512];

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  va_list args;
  va_start(args, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, args);
  va_end(args);
  return code;
}

int hip_status(hipError_t err, const char* what) {
  if (err == hipSuccess) return LLMOPT_OK;
  return fail(LLMOPT_ERR_HIP, "%s: %s", what, hipGetErrorString(err));
}

bool valid_dtype(int dt) { return dt == LLMOPT_DTYPE_F32 || dt == LLMOPT_DTYPE_F16 || dt == LLMOPT_DTYPE_BF16; }

bool aligned(const void* p, int64_t bytes) { return int64_t(reinterpret_cast<uintptr_t>(p) % uintptr_t(bytes)) == 0; }

constexpr int64_t kMaxInt = 0x7FFFFFFF;

int64_t groups(int64_t n) { return (n + kF8Group - 1) / kF8Group; }

// A matrix of rows x cols elements with `ld` elements a row (and what the name says it is).
int check_rows(const char* what, const void* p, int64_t rows, int64_t cols, int64_t ld) {
  if (rows < 0 || cols < 0) return fail(LLMOPT_ERR_INVALID_ARG, "%s: negative shape %lld x %lld", what, (long long)rows, (long long)cols);
  if (rows > kMaxInt || cols > kMaxInt) return fail(LLMOPT_ERR_UNSUPPORTED, "%s: %lld x %lld is too large", what, (long long)rows, (long long)cols);
  if (rows > 1 && ld < cols) return fail(LLMOPT_ERR_INVALID_ARG, "%s: rows of %lld elements at a stride of %lld", what, (long long)cols, (long long)ld);
  if (rows > 0 && cols > 0 && !p) return fail(LLMOPT_ERR_INVALID_ARG, "%s is null", what);
  return LLMOPT_OK;
}

#define CHECK(call)                          \
  do {                                       \
    const int rc_ = (call);                  \
    if (rc_ != LLMOPT_OK) return rc_;        \
  } while (0)

// Whether rows of codes are what the tiled kernels read: whole 16-byte pieces, and offsets within a tile in 32 bits.
bool tiled_rows(const void* p, int64_t ld, int64_t cols) {
  return aligned(p, 16) && ld % 16 == 0 && cols % 16 == 0 && ld <= (int64_t(1) << 21) && cols > 0;
}

// Workgroups of a grid of `a` x `b`.
int check_grid(int64_t a, int64_t b) {
  if (a > 0 && b > kMaxInt / a) return fail(LLMOPT_ERR_UNSUPPORTED, "%lld x %lld workgroups are too many", (long long)a, (long long)b);
  return LLMOPT_OK;
}

}  // namespace

extern "C" {

const char* llmopt_f8_last_error(void) { return g_error; }

int llmopt_f8_quantize(const void* x, int64_t ldx, int dtype, int64_t rows, int64_t cols, int64_t block_rows,
                       void* codes, int64_t ldc, void* scales, int64_t lds, void* stream) {
  if (!valid_dtype(dtype)) return fail(LLMOPT_ERR_INVALID_ARG, "bad dtype code %d", dtype);
  if (block_rows != 1 && block_rows != kF8Group)
    return fail(LLMOPT_ERR_INVALID_ARG, "a scale covers 1 or %d rows, not %lld", kF8Group, (long long)block_rows);
  CHECK(check_rows("x", x, rows, cols, ldx));
  CHECK(check_rows("codes", codes, rows, cols, ldc));
  CHECK(check_rows("scales", scales, block_rows == 1 ? rows : groups(rows), groups(cols), lds));
  CHECK(check_grid(block_rows == 1 ? rows : groups(rows), groups(cols)));
  const int64_t size = dtype == LLMOPT_DTYPE_F32 ? 4 : 2;
  F8QuantArgs a{x, ldx, static_cast<uint8_t*>(codes), ldc, static_cast<uint8_t*>(scales), lds, rows, cols, 0};
  a.vec = cols % 8 == 0 && aligned(x, 16) && (ldx * size) % 16 == 0 && aligned(codes, 8) && ldc % 8 == 0;
  return hip_status(launch_f8_quantize(a, dtype, block_rows, static_cast<hipStream_t>(stream)), "llmopt_f8_quantize");
}

int llmopt_f8_rmsnorm(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* h_out, int64_t ldh,
                      const void* weight, void* codes, int64_t ldc, void* scales, int64_t lds, int64_t rows,
                      int64_t hidden, float eps, int dtype, void* stream) {
  if (!valid_dtype(dtype)) return fail(LLMOPT_ERR_INVALID_ARG, "bad dtype code %d", dtype);
  if (dtype == LLMOPT_DTYPE_F32) return fail(LLMOPT_ERR_UNSUPPORTED, "the norm takes fp16 and bf16");
  CHECK(check_rows("x", x, rows, hidden, ldx));
  if (residual) {
    CHECK(check_rows("residual", residual, rows, hidden, ldr));
    CHECK(check_rows("h_out", h_out, rows, hidden, ldh));
  }
  CHECK(check_rows("weight", weight, 1, hidden, hidden));
  CHECK(check_rows("codes", codes, rows, hidden, ldc));
  CHECK(check_rows("scales", scales, rows, groups(hidden), lds));
  F8NormArgs a{x, ldx, residual, ldr, h_out, ldh, weight, static_cast<uint8_t*>(codes), ldc, static_cast<uint8_t*>(scales), lds, rows, hidden, eps, 0};
  auto rows16 = [](const void* p, int64_t ld) { return aligned(p, 16) && ld % 8 == 0; };
  a.vec = hidden % 8 == 0 && rows16(x, ldx) && (!residual || (rows16(residual, ldr) && rows16(h_out, ldh))) &&
          aligned(weight, 16) && aligned(codes, 8) && ldc % 8 == 0;
  return hip_status(launch_f8_rmsnorm(a, dtype, static_cast<hipStream_t>(stream)), "llmopt_f8_rmsnorm");
}

size_t llmopt_f8_linear_workspace(int64_t M, int64_t N, int64_t K) {
  (void)M, (void)N, (void)K;
  return 0;
}

int llmopt_f8_linear(const void* x, int64_t ldx, const void* x_scales, int64_t ldxs, int64_t M, int64_t K,
                     const void* w, int64_t ldw, const void* w_scales, int64_t ldws, const void* bias, void* y,
                     int64_t ldy, int64_t N, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  (void)workspace, (void)workspace_bytes;
  if (!valid_dtype(out_dtype)) return fail(LLMOPT_ERR_INVALID_ARG, "bad dtype code %d", out_dtype);
  if (out_dtype == LLMOPT_DTYPE_F32) return fail(LLMOPT_ERR_UNSUPPORTED, "the product is fp16 or bf16");
  CHECK(check_rows("x", x, M, K, ldx));
  CHECK(check_rows("x_scales", x_scales, M, groups(K), ldxs));
  CHECK(check_rows("w", w, N, K, ldw));
  CHECK(check_rows("w_scales", w_scales, groups(N), groups(K), ldws));
  CHECK(check_rows("y", y, M, N, ldy));
  CHECK(check_grid((M + 15) / 16, (N + 63) / 64));
  if (M > 64 && tiled_rows(x, ldx, K) && tiled_rows(w, ldw, K)) {
    F8TilesArgs t{};
    t.x = static_cast<const uint8_t*>(x);
    t.ldx = ldx;
    t.x_scales = static_cast<const uint8_t*>(x_scales);
    t.ldxs = ldxs;
    t.w[0] = {static_cast<const uint8_t*>(w), ldw, static_cast<const uint8_t*>(w_scales), ldws};
    t.bias = bias;
    t.y = y;
    t.ldy = ldy;
    t.M = M, t.N = N, t.K = K;
    t.splits = 1;
    t.vec = aligned(y, 16) && ldy % 8 == 0;
    return hip_status(launch_f8_tiles(t, F8Shape::k256x256, out_dtype, static_cast<hipStream_t>(stream)), "llmopt_f8_linear");
  }
  const F8LinearArgs a{static_cast<const uint8_t*>(x), ldx, static_cast<const uint8_t*>(x_scales), ldxs, {static_cast<const uint8_t*>(w), ldw, static_cast<const uint8_t*>(w_scales), ldws},
                       bias, y, ldy, M, N, K};
  return hip_status(launch_f8_linear_any(a, out_dtype, static_cast<hipStream_t>(stream)), "llmopt_f8_linear");
}

size_t llmopt_f8_swiglu_workspace(int64_t M, int64_t N, int64_t K) {
  (void)K;
  return M > 0 && N > 0 ? size_t(M) * size_t((N + 7) / 8 * 8) * 2 * sizeof(float) : 0;
}

int llmopt_f8_swiglu(const void* x, int64_t ldx, const void* x_scales, int64_t ldxs, int64_t M, int64_t K,
                     const void* gate, int64_t ldg, const void* gate_scales, int64_t ldgs, const void* up, int64_t ldu,
                     const void* up_scales, int64_t ldus, int64_t N, void* codes, int64_t ldc, void* scales,
                     int64_t lds, void* workspace, size_t workspace_bytes, void* stream) {
  CHECK(check_rows("x", x, M, K, ldx));
  CHECK(check_rows("x_scales", x_scales, M, groups(K), ldxs));
  CHECK(check_rows("gate", gate, N, K, ldg));
  CHECK(check_rows("gate_scales", gate_scales, groups(N), groups(K), ldgs));
  CHECK(check_rows("up", up, N, K, ldu));
  CHECK(check_rows("up_scales", up_scales, groups(N), groups(K), ldus));
  CHECK(check_rows("codes", codes, M, N, ldc));
  CHECK(check_rows("scales", scales, M, groups(N), lds));
  CHECK(check_grid((M + 15) / 16, (N + 63) / 64));
  CHECK(check_grid(M, groups(N)));
  if (M == 0 || N == 0) return LLMOPT_OK;
  if (M > 64 && tiled_rows(x, ldx, K) && tiled_rows(gate, ldg, K) && tiled_rows(up, ldu, K)) {
    F8TilesArgs t{};
    t.x = static_cast<const uint8_t*>(x);
    t.ldx = ldx;
    t.x_scales = static_cast<const uint8_t*>(x_scales);
    t.ldxs = ldxs;
    t.w[0] = {static_cast<const uint8_t*>(gate), ldg, static_cast<const uint8_t*>(gate_scales), ldgs};
    t.w[1] = {static_cast<const uint8_t*>(up), ldu, static_cast<const uint8_t*>(up_scales), ldus};
    t.codes = static_cast<uint8_t*>(codes);
    t.ldc = ldc;
    t.scales = static_cast<uint8_t*>(scales);
    t.lds = lds;
    t.M = M, t.N = N, t.K = K;
    t.splits = 1;
    t.vec = aligned(codes, 16) && ldc % 16 == 0;
    return hip_status(launch_f8_tiles(t, F8Shape::k256x256, 0, static_cast<hipStream_t>(stream)), "llmopt_f8_swiglu");
  }
  const size_t need = llmopt_f8_swiglu_workspace(M, N, K);
  if (workspace_bytes < need || (need && !workspace) || !aligned(workspace, 16))
    return fail(LLMOPT_ERR_WORKSPACE, "llmopt_f8_swiglu needs %zu bytes of workspace, aligned to 16", need);
  const int64_t ld = (N + 7) / 8 * 8;
  float* sums = static_cast<float*>(workspace);
  F8LinearArgs a{static_cast<const uint8_t*>(x), ldx, static_cast<const uint8_t*>(x_scales), ldxs, {static_cast<const uint8_t*>(gate), ldg, static_cast<const uint8_t*>(gate_scales), ldgs},
                 nullptr, sums, ld, M, N, K};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  CHECK(hip_status(launch_f8_linear_any(a, LLMOPT_DTYPE_F32, st), "llmopt_f8_swiglu"));
  a.w = {static_cast<const uint8_t*>(up), ldu, static_cast<const uint8_t*>(up_scales), ldus};
  a.y = sums + M * ld;
  CHECK(hip_status(launch_f8_linear_any(a, LLMOPT_DTYPE_F32, st), "llmopt_f8_swiglu"));
  const F8ActArgs act{sums, sums + M * ld, ld, static_cast<uint8_t*>(codes), ldc, static_cast<uint8_t*>(scales), lds, M, N};
  return hip_status(launch_f8_act(act, st), "llmopt_f8_swiglu");
}

}  // extern "C"
