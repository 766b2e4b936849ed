// C ABI of llmopt_float8.h: checks, the choice of kernels, and launches.
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>

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

// Whether rows of codes are what the decode and tiled kernels read: whole 16-byte pieces, and offsets within a tile in 32 bits
// (those of a row's scales, too).
bool tiled_rows(const void* p, int64_t ld, int64_t cols, int64_t ld_scales = 0) {
  constexpr int64_t kMost = int64_t(1) << 21;
  return aligned(p, 16) && ld % 16 == 0 && cols % 16 == 0 && ld <= kMost && cols > 0 && cols <= kMost && ld_scales <= kMost;
}

// The stride of `rows` rows of codes. A single row has any: its length, then, so that the rows behind it, whose positions the tiles take
// from the stride, lie behind the operand's end.
int64_t stride_of(int64_t rows, int64_t cols, int64_t ld) { return rows == 1 ? cols : ld; }

// Workgroups of a grid of `a` x `b`.
int check_grid(int64_t a, int64_t b, int64_t most = kMaxInt) {
  if (a > 0 && b > most / a) return fail(LLMOPT_ERR_UNSUPPORTED, "%lld x %lld workgroups are too many", (long long)a, (long long)b);
  return LLMOPT_OK;
}

// Workgroups of 256 threads of the kernels for any rows: work-items are counted in 32 bits. (Outputs of 2^34.)
constexpr int64_t kMostAny = (int64_t(1) << 24) - 1;

// ---- the choice of kernels --------------------------------------------------------------------------

constexpr int64_t kFewTokens = 16;  // that the decode kernel takes of any weight
constexpr int64_t kSomeTokens = 1024;  // that it takes at most, 32 at a time

// The decode kernel, or a tile's shape and the parts of K: the least of an estimate of the time. A workgroup's step of 128 columns takes
// `alone` us where few workgroups run and `full` where every CU has its share; a round of workgroups (256 of them, or 512 where two
// fit a CU) adds `round`, the first loads and the results; parts are written and read again at some 3 TB/s. Over 97 sizes, two
// thirds of them drawn at random (17 to 1024 tokens, 128 to 10240 features and columns), the choice takes 0.8 % more than the best of all on
// average and 17 % at most; over 120 of 1500 to 8192 tokens (1024 to 6144 features, 256 to 4096 columns) 1.4 % and 11 %, nearly all of
// it at up to 1024 columns, where 128 x 128 is faster than 256 x 256; over 47 gated ones of 17 to 8192 tokens 0.8 %, and 32 % at
// most (9000 x 3600, 25 tokens: 256 x 64 41, the decode kernel 31).
// Measured (MI355X, in a graph, us; the estimate's choice first): 4096 x 14336, 8192 tokens, 256 x 256 377, 256 x 128 441, 256 x
// 64 593; 1024 tokens, 256 x 128 in two parts 74, 256 x 64 88, 256 x 256 161; 32 tokens, 128 x 64 in eight parts 18.6, whole 57, the
// decode kernel 19.6; 6144 x 4096, 200 tokens, 128 x 64 20, 256 x 64 27, 256 x 256 52; 17 tokens, the decode kernel 12.5, 128 x 64 in eight
// parts 14.1; 1536 x 1040, 777 tokens, 128 x 64 9.8, 128 x 128 12, 256 x 256 21; 1536 x 1024, 8192 tokens, 256 x 256 25.3, 128 x
// 128 23.9; gate and up 2816 x 1024, 32 tokens, the decode kernel 8.6, 256 x 64 12.1.
struct Tile {
  F8Shape shape;
  int64_t n, m, per_cu;
  double alone, full, round;
};
constexpr Tile kTiles[] = {
    {F8Shape::k256x256, 256, 256, 1, 1.38, 1.62, 5.0}, {F8Shape::k256x128, 256, 128, 1, 0.78, 0.93, 4.0},
    {F8Shape::k256x64, 256, 64, 1, 0.75, 0.72, 3.0},   {F8Shape::k128x128, 128, 128, 2, 0.94, 1.07, 3.5},
    {F8Shape::k128x64, 128, 64, 2, 0.50, 0.76, 3.0},
};

struct Plan {
  F8Shape shape;
  int64_t splits, steps_per_split;
  bool few;  // the decode kernel instead (gated: with the sums in the workspace)
};

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t padded(int64_t n) { return up(n, 16) * 16; }

size_t sums_bytes(int64_t M, int64_t N) { return size_t(2) * size_t(M) * size_t(padded(N)) * sizeof(float); }

// The decode kernel's time over tiles of 32 tokens, and the gated product's second launch. One workgroup fits a CU, two where a
// row has at most 16 steps.
double decode_us(int64_t M, int64_t N, int64_t steps, bool gated) {
  const int64_t count = up(N, 16) * (gated ? 2 : 1) * up(M, 32), held = steps > 16 ? 256 : 512;
  const double load = std::min(1.0, double(count) / double(held));
  const double step = 0.04 + (steps > 16 ? 0.06 : 0.13) * load + 0.05 * double(std::min<int64_t>(M, 32)) / 32.0;
  return 2.0 + double(up(count, held)) * (1.0 + double(steps) * step) + (gated ? 2.0 + double(M) * double(N) * 9.0 / 4e6 : 0.0);
}

size_t parts_bytes(int64_t M, int64_t N, int64_t splits) {
  return splits > 1 ? size_t(splits) * size_t(M) * size_t(padded(N)) * sizeof(float) : 0;
}

Plan plan_tiles(int64_t M, int64_t N, int64_t K, bool gated, size_t workspace) {
  Plan best{F8Shape::k256x256, 1, 1, false};
  double least = 1e30;
  const int64_t steps = std::max<int64_t>(1, groups(K));
  const bool room = !gated || workspace >= sums_bytes(M, N);
  if (room && M <= kFewTokens) return Plan{F8Shape::k256x256, 1, steps, true};
  if (room && M <= kSomeTokens) least = decode_us(M, N, steps, gated), best.few = true;
  for (const Tile& t : kTiles) {
    if (gated && t.n != 256) continue;  // a group of 128 features of both weights
    const int64_t tiles = up(N, gated ? t.n / 2 : t.n) * up(M, t.m);
    const int64_t most = gated || t.m == 256 ? 1 : 8;  // (with tiles this large there are smaller ones in fewer parts)
    for (int64_t splits = 1; splits <= most; splits *= 2) {
      const int64_t per = up(steps, splits);
      if (splits > 1 && (per < 4 || up(steps, per) != splits || parts_bytes(M, N, splits) > workspace)) break;
      const int64_t count = tiles * splits, rounds = up(count, 256 * t.per_cu);
      const double load = std::clamp(double(count) / 256.0 - double(t.per_cu - 1), 0.0, 1.0);
      double us = double(rounds) * (double(per) * (t.alone + (t.full - t.alone) * load) + t.round) + 2.0;
      if (splits > 1) us += 3.0 + double(M) * double(N) * 8.0 * double(splits) / 3e6;
      if (us < least) least = us, best = Plan{t.shape, splits, per, false};
    }
  }
  return best;
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
  if (M < 1 || N < 1 || K < 1 || M > kMaxInt || N > kMaxInt || K > kMaxInt) return 0;
  const Plan plan = plan_tiles(M, N, K, false, SIZE_MAX);
  return plan.few ? 0 : parts_bytes(M, N, plan.splits);
}

int llmopt_f8_linear(const void* x, int64_t ldx, const void* x_scales, int64_t ldxs, int64_t M, int64_t K,
                     const void* w, int64_t ldw, const void* w_scales, int64_t ldws, const void* bias, void* y,
                     int64_t ldy, int64_t N, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_dtype(out_dtype)) return fail(LLMOPT_ERR_INVALID_ARG, "bad dtype code %d", out_dtype);
  if (out_dtype == LLMOPT_DTYPE_F32) return fail(LLMOPT_ERR_UNSUPPORTED, "the product is fp16 or bf16");
  CHECK(check_rows("x", x, M, K, ldx));
  CHECK(check_rows("x_scales", x_scales, M, groups(K), ldxs));
  CHECK(check_rows("w", w, N, K, ldw));
  CHECK(check_rows("w_scales", w_scales, groups(N), groups(K), ldws));
  CHECK(check_rows("y", y, M, N, ldy));
  CHECK(check_grid(8 * up(M, 16), up(N, 64)));
  if (M == 0 || N == 0) return LLMOPT_OK;
  ldx = stride_of(M, K, ldx), ldw = stride_of(N, K, ldw);
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
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (!tiled_rows(x, ldx, K, ldxs) || !tiled_rows(w, ldw, K)) {
    CHECK(check_grid(up(M, 16), up(N, 64), kMostAny));
    return hip_status(launch_f8_any(t, out_dtype, st), "llmopt_f8_linear");
  }
  const Plan plan = plan_tiles(M, N, K, false, workspace && aligned(workspace, 16) ? workspace_bytes : 0);
  if (plan.few) {
    const F8DecodeArgs d{t.x, ldx, t.x_scales, ldxs, {t.w[0], {}}, bias, y, ldy, M, N, K, 0, 0};
    return hip_status(launch_f8_decode(d, out_dtype, st), "llmopt_f8_linear");
  }
  t.splits = uint32_t(plan.splits);
  t.steps_per_split = uint32_t(plan.steps_per_split);
  t.parts = static_cast<float*>(workspace);
  t.ld_parts = padded(N);
  return hip_status(launch_f8_tiles(t, plan.shape, out_dtype, st), "llmopt_f8_linear");
}

size_t llmopt_f8_swiglu_workspace(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1 || M > kMaxInt || N > kMaxInt || K > kMaxInt) return 0;
  return plan_tiles(M, N, K, true, SIZE_MAX).few ? sums_bytes(M, N) : 0;
}

int llmopt_f8_swiglu(const void* x, int64_t ldx, const void* x_scales, int64_t ldxs, int64_t M, int64_t K,
                     const void* gate, int64_t ldg, const void* gate_scales, int64_t ldgs, const void* up_, int64_t ldu,
                     const void* up_scales, int64_t ldus, int64_t N, void* codes, int64_t ldc, void* scales,
                     int64_t lds, void* workspace, size_t workspace_bytes, void* stream) {
  CHECK(check_rows("x", x, M, K, ldx));
  CHECK(check_rows("x_scales", x_scales, M, groups(K), ldxs));
  CHECK(check_rows("gate", gate, N, K, ldg));
  CHECK(check_rows("gate_scales", gate_scales, groups(N), groups(K), ldgs));
  CHECK(check_rows("up", up_, N, K, ldu));
  CHECK(check_rows("up_scales", up_scales, groups(N), groups(K), ldus));
  CHECK(check_rows("codes", codes, M, N, ldc));
  CHECK(check_rows("scales", scales, M, groups(N), lds));
  CHECK(check_grid(up(M, 16), up(N, 64)));
  if (M == 0 || N == 0) return LLMOPT_OK;
  ldx = stride_of(M, K, ldx), ldg = stride_of(N, K, ldg), ldu = stride_of(N, K, ldu);
  F8TilesArgs t{};
  t.x = static_cast<const uint8_t*>(x);
  t.ldx = ldx;
  t.x_scales = static_cast<const uint8_t*>(x_scales);
  t.ldxs = ldxs;
  t.w[0] = {static_cast<const uint8_t*>(gate), ldg, static_cast<const uint8_t*>(gate_scales), ldgs};
  t.w[1] = {static_cast<const uint8_t*>(up_), ldu, static_cast<const uint8_t*>(up_scales), ldus};
  t.codes = static_cast<uint8_t*>(codes);
  t.ldc = ldc;
  t.scales = static_cast<uint8_t*>(scales);
  t.lds = lds;
  t.M = M, t.N = N, t.K = K;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // Without columns a weight has no codes to point to.
  if (K == 0) t.w[0].codes = t.w[1].codes = static_cast<const uint8_t*>(codes);
  if (!tiled_rows(x, ldx, K, ldxs) || !tiled_rows(gate, ldg, K) || !tiled_rows(up_, ldu, K)) {
    CHECK(check_grid(up(M, 16), up(N, 64), kMostAny));
    return hip_status(launch_f8_any(t, 0, st), "llmopt_f8_swiglu");
  }
  const Plan plan = plan_tiles(M, N, K, true, workspace && aligned(workspace, 16) ? workspace_bytes : 0);
  if (plan.few) {
    float* sums = static_cast<float*>(workspace);
    const int64_t ld = padded(N);
    const F8DecodeArgs d{t.x, ldx, t.x_scales, ldxs, {t.w[0], t.w[1]}, nullptr, sums, ld, M, N, K, 0, 0};
    CHECK(hip_status(launch_f8_decode(d, kDtF32, st), "llmopt_f8_swiglu"));
    const F8ActArgs act{{t.x, ldx, t.x_scales, ldxs, {t.w[0], t.w[1]}, K}, sums, sums + M * ld, ld, t.codes, ldc, t.scales, lds, M, N};
    return hip_status(launch_f8_act(act, st), "llmopt_f8_swiglu");
  }
  t.splits = 1;
  return hip_status(launch_f8_tiles(t, plan.shape, 0, st), "llmopt_f8_swiglu");
}

}  // extern "C"
