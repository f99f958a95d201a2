// C ABI of the gfx950 ConvRot library (declared in include/convrot_amd.h).
//
// Every entry point validates its arguments before any launch and reports
// failures as a status code plus a thread-local message; messages for the
// conditions the reference checks reuse the reference's wording
// (/root/reference/src/convrot_mlx/core.py:50-61,75-77,431-442,1030-1058).
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <atomic>

#include "convrot_launch.h"
#include "gemm_groups.h"

namespace convrot {
namespace {
// Tuning overrides, stored as value + 1 so that the zero-initialized table
// means "nothing set".
std::atomic<int> g_tuning[kTuneCount] = {};
}  // namespace

int tuning(TuneKey key) { return g_tuning[key].load(std::memory_order_relaxed) - 1; }
}  // namespace convrot

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int ok() {
  g_err[0] = '\0';
  return CONVROT_OK;
}

int launch_status(hipError_t e, const char* what) {
  if (e != hipSuccess) return fail(CONVROT_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return ok();
}

bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p % a) == 0; }

bool valid_dtype(int dt) { return dt == CONVROT_DTYPE_F32 || dt == CONVROT_DTYPE_F16 || dt == CONVROT_DTYPE_BF16; }

const char* dtype_name(int dt) {
  switch (dt) {
    case CONVROT_DTYPE_F32: return "float32";
    case CONVROT_DTYPE_F16: return "float16";
    case CONVROT_DTYPE_BF16: return "bfloat16";
    default: return "unknown";
  }
}

// core.py:50-61; returns log4(G) or -1
int log4_group(int g) {
  if (g < 4) return -1;
  int s = 0;
  while (g > 1 && g % 4 == 0) {
    g /= 4;
    ++s;
  }
  return g == 1 ? s : -1;
}

constexpr int64_t kMaxFeatures = 65536;
// The GEMM kernels address the packed weights ([ceil(K/128)][ceil(N/16)][1 KB])
// through buffer resources with 32-bit signed offsets: below 2 GiB.
constexpr int64_t kMaxWeightBytes = int64_t(1) << 31;
int64_t packed_weight_bytes(int64_t N, int64_t K) { return ((K + 127) / 128) * ((N + 15) / 16) * 1024; }
// The FP6 GEMM reads each operand through one buffer resource: 32-bit offsets
// (a k-block's offset plus a tile's pieces) must not wrap, so an operand stays
// 1 MiB below 4 GiB.
constexpr int64_t kMaxFp6OperandBytes = (int64_t(1) << 32) - (int64_t(1) << 20);

}  // namespace

extern "C" {

const char* convrot_last_error(void) { return g_err; }

int convrot_set_tuning(const char* name, const char* value) {
  using namespace convrot;
  if (!name) return fail(CONVROT_ERR_INVALID, "null tuning name");
  static const struct {
    const char* name;
    TuneKey key;
  } kNames[] = {{"gemm_tile", kTuneGemmTile},         {"gemm_sk", kTuneGemmSk},
                {"gemm_sk_min", kTuneGemmSkMin},      {"gemm_no_dma", kTuneGemmNoDma},
                {"gemm_smallm_max", kTuneGemmSmallmMax}, {"w4a4_smallm_cfg", kTuneW4a4SmallmCfg},
                {"w4a16_cfg", kTuneW4a16Cfg},         {"w4a16_tile", kTuneW4a16Tile},
                {"prep_ni", kTunePrepNi},             {"sk_spin_limit", kTuneSkSpinLimit},
                {"gemm_persist", kTuneGemmPersist},   {"gemm_mfma32", kTuneGemmMfma32},
                {"fp6_tile", kTuneFp6Tile},           {"linear_rows_cfg", kTuneRowsCfg},
                {"w4a4_midm_cfg", kTuneMidmCfg},      {"fp6_split", kTuneFp6Split},
                {"w8a8_tile", kTuneW8a8Tile},         {"w8a8_split", kTuneW8a8Split},
                {"fp8_tile", kTuneFp8Tile},           {"fp8_split", kTuneFp8Split},
                {"grouped_tile", kTuneGroupedTile}};
  int key = -1;
  for (const auto& n : kNames)
    if (strcmp(n.name, name) == 0) key = n.key;
  if (key < 0) return fail(CONVROT_ERR_INVALID, "unknown tuning override '%s'", name);
  int v = -1;
  if (value && value[0]) {
    bool good = true;
    switch (key) {
      case kTuneGemmTile: {
        int bm = 0, bn = 0, wm = 2, wn = 2, st = 0;
        const int got = sscanf(value, "%dx%dw%dx%ds%d", &bm, &bn, &wm, &wn, &st);
        good = got >= 2 && bm > 0 && bm <= 512 && bn > 0 && bn <= 512 && wm > 0 && wm < 16 && wn > 0 && wn < 16 &&
               st >= 0 && st < 8 && w4a4_tile_known(bm, bn, wm, wn, st);
        v = bm | bn << 10 | wm << 20 | wn << 24 | st << 28;
        break;
      }
      case kTuneFp6Tile:
      case kTuneW8a8Tile:
      case kTuneFp8Tile:
      case kTuneGroupedTile:
      case kTuneW4a16Tile: {
        int bm = 0, bn = 0;
        char tail = 0;
        good = sscanf(value, "%dx%d%c", &bm, &bn, &tail) == 2 &&
               (key == kTuneFp6Tile    ? fp6_tile_known(bm, bn)
                : key == kTuneW8a8Tile ? w8a8_tile_known(bm, bn)
                : key == kTuneFp8Tile  ? fp8_tile_known(bm, bn)
                : key == kTuneGroupedTile ? grouped_tile_known(bm, bn)
                                       : w4a16_tile_known(bm, bn));
        v = bm | bn << 10;
        break;
      }
      case kTuneW4a4SmallmCfg:
        good = strchr("ABCF", value[0]) != nullptr && value[1] == '\0';
        v = value[0];
        break;
      case kTuneW4a16Cfg:
        good = strchr("ABCDEFST", value[0]) != nullptr && value[1] == '\0';
        v = value[0];
        break;
      case kTuneRowsCfg:
        v = atoi(value);
        good = v == 1 || v == 2 || v == 3 || v == 5 || v == 16;
        break;
      case kTuneFp6Split:
        v = atoi(value);
        good = v == 1 || v == 2 || v == 4;
        break;
      case kTuneW8a8Split:
      case kTuneFp8Split:
        v = atoi(value);
        good = v >= 1 && v <= 64;
        break;
      case kTuneMidmCfg:
        v = atoi(value);
        good = midm_split_known(v);
        break;
      default: {
        char* end = nullptr;
        const long long n = strtoll(value, &end, 10);
        good = end && *end == '\0' && n >= 0 && n <= 0x7fffffff;
        v = (int)n;
      }
    }
    if (!good) return fail(CONVROT_ERR_INVALID, "invalid value '%s' for tuning override '%s'", value, name);
  }
  g_tuning[key].store(v + 1, std::memory_order_relaxed);
  return ok();
}

const char* convrot_version(void) { return "convrot-mi355x 0.1.0 (gfx950)"; }

int64_t convrot_cdna4_bytes(int64_t N, int64_t K) {
  if (N < 0 || K < 0) return -1;
  return ((K + 127) / 128) * ((N + 15) / 16) * 1024;
}

int64_t convrot_fp6_bytes(int64_t R, int64_t K) {
  if (R < 0 || K < 0 || K % 128) return -1;
  return (K / 128) * ((R + 15) / 16) * 1536;
}

int convrot_w4a4_blocked(int64_t M, int64_t N, int64_t K) { return convrot::midm_preferred(M, N, K) ? 1 : 0; }

int convrot_w4a4_fp6_tile(int64_t M, int64_t N, int* bm, int* bn) {
  if (M <= 0 || N <= 0 || !bm || !bn)
    return fail(CONVROT_ERR_INVALID, "FP6 tile query needs M, N > 0 and two result pointers");
  convrot::fp6_plan_tile(M, N, bm, bn);
  return ok();
}

int convrot_w4a4_fp6_compact_tile(int64_t M, int64_t N, int* bm, int* bn, int* parts) {
  if (M <= 0 || N <= 0 || !bm || !bn || !parts)
    return fail(CONVROT_ERR_INVALID, "compact FP6 tile query needs M, N > 0 and three result pointers");
  convrot::fp6_plan_compact(M, N, bm, bn, parts);
  return ok();
}

int convrot_prepare_plan(int64_t rows, int64_t features, int dtype, int group_size, int mode, int producer,
                         int* iterations, int* waves, int* packed) {
  const bool no_rotate = (mode & CONVROT_PREP_NO_ROTATE) != 0;
  const int kind = mode & ~CONVROT_PREP_NO_ROTATE, s = no_rotate ? 0 : log4_group(group_size);
  if (rows < 0 || features <= 0 || features > kMaxFeatures || !valid_dtype(dtype) || s < 0 || s > 5 ||
      kind < CONVROT_PREP_PACKED || kind > CONVROT_PREP_INT8_BLOCKED || producer < CONVROT_PRODUCER_PLAIN ||
      producer > CONVROT_PRODUCER_GELU || !iterations || !waves || !packed)
    return fail(CONVROT_ERR_INVALID, "preparation plan query: bad shape, dtype, group, mode, producer or result pointer");
  bool p = false;
  if (!convrot::prep_route(rows, features, dtype, s, kind, producer, iterations, waves, &p))
    return fail(CONVROT_ERR_UNSUPPORTED, "no preparation plan for %lld features", (long long)features);
  *packed = p ? 1 : 0;
  return ok();
}

int convrot_prepare(const void* x, int dtype, int64_t rows, int64_t features, int group_size, int mode,
                    void* out, float* scales, void* stream) {
  const bool no_rotate = (mode & CONVROT_PREP_NO_ROTATE) != 0;
  const int kind = mode & ~CONVROT_PREP_NO_ROTATE;
  if (kind != CONVROT_PREP_PACKED && kind != CONVROT_PREP_INT8 && kind != CONVROT_PREP_ROTATE &&
      kind != CONVROT_PREP_FP6 && kind != CONVROT_PREP_INT8_BLOCKED)
    return fail(CONVROT_ERR_INVALID, "unknown ConvRot preparation mode %d", mode);
  if (kind == CONVROT_PREP_FP6 && features % 128)
    return fail(CONVROT_ERR_UNSUPPORTED, "FP6 preparation requires features divisible by 128, got %lld",
                (long long)features);
  if (no_rotate && kind == CONVROT_PREP_ROTATE)
    return fail(CONVROT_ERR_INVALID, "rotate mode cannot skip the rotation");
  if (!valid_dtype(dtype)) return fail(CONVROT_ERR_INVALID, "unsupported activation dtype code %d", dtype);
  if (rows < 0 || features <= 0) return fail(CONVROT_ERR_INVALID, "invalid shape (%lld, %lld)", (long long)rows, (long long)features);
  int s = 0;
  if (!no_rotate) {
    s = log4_group(group_size);
    if (s < 0) return fail(CONVROT_ERR_INVALID, "Regular Hadamard size must be a power of 4, got %d", group_size);
    if (s > 5)
      return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot supports groups [4, 16, 64, 256, 1024], got %d", group_size);
    if (features % group_size)
      return fail(CONVROT_ERR_INVALID, "features %lld not divisible by ConvRot group size %d", (long long)features,
                  group_size);
  }
  if (features % 16)
    return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot preparation requires features divisible by 16, got %lld",
                (long long)features);
  if (features > kMaxFeatures)
    return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot preparation supports at most %lld features, got %lld",
                (long long)kMaxFeatures, (long long)features);
  if (rows > 0x7fffffff) return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot preparation supports at most 2^31-1 rows");
  if (rows == 0) return ok();
  if (!x || !out || (kind != CONVROT_PREP_ROTATE && !scales))
    return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(x, 16) || !aligned(out, 16)) return fail(CONVROT_ERR_INVALID, "x and out must be 16-byte aligned");
  return launch_status(convrot::launch_prep(x, dtype, rows, features, s, kind, out, scales, (hipStream_t)stream),
                       "convrot_prepare");
}

int convrot_prepare_modulated(const void* x, int dtype, int64_t rows, int64_t features, int group_size, int mode,
                              const void* shift, const void* scale, int64_t rows_per_vector, float eps, void* out,
                              float* scales, void* stream) {
  if (mode & CONVROT_PREP_NO_ROTATE)
    return fail(CONVROT_ERR_INVALID, "the modulated producer always rotates (no CONVROT_PREP_NO_ROTATE)");
  if (mode != CONVROT_PREP_PACKED && mode != CONVROT_PREP_INT8 && mode != CONVROT_PREP_ROTATE &&
      mode != CONVROT_PREP_FP6 && mode != CONVROT_PREP_INT8_BLOCKED)
    return fail(CONVROT_ERR_INVALID, "unknown ConvRot preparation mode %d", mode);
  if (!valid_dtype(dtype)) return fail(CONVROT_ERR_INVALID, "unsupported activation dtype code %d", dtype);
  if (rows < 0 || features <= 0) return fail(CONVROT_ERR_INVALID, "invalid shape (%lld, %lld)", (long long)rows, (long long)features);
  if (rows_per_vector <= 0 || rows_per_vector > 0x7fffffff)
    return fail(CONVROT_ERR_INVALID, "rows_per_vector must be in [1, 2^31-1], got %lld", (long long)rows_per_vector);
  if (!(eps >= 0.0f) || eps > 1e30f) return fail(CONVROT_ERR_INVALID, "eps must be finite and non-negative");
  const int s = log4_group(group_size);
  if (s < 0) return fail(CONVROT_ERR_INVALID, "Regular Hadamard size must be a power of 4, got %d", group_size);
  if (s > 5) return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot supports groups [4, 16, 64, 256, 1024], got %d", group_size);
  if (features % group_size)
    return fail(CONVROT_ERR_INVALID, "features %lld not divisible by ConvRot group size %d", (long long)features, group_size);
  if (mode == CONVROT_PREP_FP6 && features % 128)
    return fail(CONVROT_ERR_UNSUPPORTED, "FP6 preparation requires features divisible by 128, got %lld",
                (long long)features);
  if (features % 16)
    return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot preparation requires features divisible by 16, got %lld",
                (long long)features);
  if (features > kMaxFeatures)
    return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot preparation supports at most %lld features, got %lld",
                (long long)kMaxFeatures, (long long)features);
  if (rows > 0x7fffffff) return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot preparation supports at most 2^31-1 rows");
  if (rows == 0) return ok();
  if (!x || !out || !shift || !scale || (mode != CONVROT_PREP_ROTATE && !scales))
    return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(x, 16) || !aligned(out, 16) || !aligned(shift, 16) || !aligned(scale, 16))
    return fail(CONVROT_ERR_INVALID, "x, out, shift and scale must be 16-byte aligned");
  return launch_status(convrot::launch_prep_modulated(x, dtype, rows, features, s, mode, shift, scale,
                                                      rows_per_vector, eps, out, scales, (hipStream_t)stream),
                       "convrot_prepare_modulated");
}

int convrot_prepare_gelu(const void* head, int64_t head_features, int64_t head_stride, const void* x,
                         int64_t x_features, int64_t x_stride, int dtype, int64_t rows, int group_size, int mode,
                         void* out, float* scales, void* stream) {
  if (mode & CONVROT_PREP_NO_ROTATE)
    return fail(CONVROT_ERR_INVALID, "the GELU producer always rotates (no CONVROT_PREP_NO_ROTATE)");
  if (mode != CONVROT_PREP_PACKED && mode != CONVROT_PREP_INT8 && mode != CONVROT_PREP_ROTATE &&
      mode != CONVROT_PREP_FP6 && mode != CONVROT_PREP_INT8_BLOCKED)
    return fail(CONVROT_ERR_INVALID, "unknown ConvRot preparation mode %d", mode);
  if (!valid_dtype(dtype)) return fail(CONVROT_ERR_INVALID, "unsupported activation dtype code %d", dtype);
  if (rows < 0 || head_features < 0 || x_features <= 0)
    return fail(CONVROT_ERR_INVALID, "invalid GELU producer shape: rows %lld, head %lld, x %lld features",
                (long long)rows, (long long)head_features, (long long)x_features);
  if (head_features % 16 || x_features % 16)
    return fail(CONVROT_ERR_UNSUPPORTED, "the GELU producer requires head and x features divisible by 16, got %lld and %lld",
                (long long)head_features, (long long)x_features);
  const int64_t features = head_features + x_features;
  const int s = log4_group(group_size);
  if (s < 0) return fail(CONVROT_ERR_INVALID, "Regular Hadamard size must be a power of 4, got %d", group_size);
  if (s > 5) return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot supports groups [4, 16, 64, 256, 1024], got %d", group_size);
  if (features % group_size)
    return fail(CONVROT_ERR_INVALID, "features %lld not divisible by ConvRot group size %d", (long long)features, group_size);
  if (mode == CONVROT_PREP_FP6 && features % 128)
    return fail(CONVROT_ERR_UNSUPPORTED, "FP6 preparation requires features divisible by 128, got %lld",
                (long long)features);
  if (features > kMaxFeatures)
    return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot preparation supports at most %lld features, got %lld",
                (long long)kMaxFeatures, (long long)features);
  if (x_stride < x_features || (head_features > 0 && head_stride < head_features))
    return fail(CONVROT_ERR_INVALID, "row strides (head %lld, x %lld) shorter than the rows", (long long)head_stride,
                (long long)x_stride);
  if (rows > 0x7fffffff) return fail(CONVROT_ERR_UNSUPPORTED, "fused ConvRot preparation supports at most 2^31-1 rows");
  if (rows == 0) return ok();
  const int64_t esize = dtype == CONVROT_DTYPE_F32 ? 4 : 2;
  if (!x || !out || (head_features > 0 && !head) || (mode != CONVROT_PREP_ROTATE && !scales))
    return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(x, 16) || !aligned(out, 16) || (head_features > 0 && !aligned(head, 16)) || (x_stride * esize) % 16 ||
      (head_features > 0 && (head_stride * esize) % 16))
    return fail(CONVROT_ERR_INVALID, "x, head and out rows must start 16-byte aligned");
  return launch_status(convrot::launch_prep_gelu(head, head_features, head_stride, x, x_features, x_stride, dtype,
                                                 rows, s, mode, out, scales, (hipStream_t)stream),
                       "convrot_prepare_gelu");
}

namespace {

// Argument checks shared by the W4A4 GEMM entry points; CONVROT_OK when the
// launch may proceed (M == 0 or N == 0 included).
int check_w4a4(const void* act, int act_format, const float* xscales, const uint8_t* qweight,
               const float* wscales, int64_t M, int64_t N, int64_t K, void* out, int out_dtype) {
  if (act_format != CONVROT_ACT_PACKED && act_format != CONVROT_ACT_INT8 && act_format != CONVROT_ACT_INT8_BLOCKED)
    return fail(CONVROT_ERR_INVALID, "unknown activation format %d", act_format);
  if (!valid_dtype(out_dtype)) return fail(CONVROT_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 0 || K <= 0) return fail(CONVROT_ERR_INVALID, "invalid GEMM shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (K % 32) return fail(CONVROT_ERR_INVALID, "W4A4 GEMM requires K divisible by 32, got %lld", (long long)K);
  if (K > kMaxFeatures)
    return fail(CONVROT_ERR_UNSUPPORTED, "W4A4 GEMM supports K up to %lld, got %lld", (long long)kMaxFeatures, (long long)K);
  if (M > 0x7fffffff || N > 0x7fffffff) return fail(CONVROT_ERR_UNSUPPORTED, "GEMM dimension too large");
  if (act_format == CONVROT_ACT_INT8_BLOCKED && ((K + 127) / 128) * ((M + 15) / 16) * 2048 >= kMaxWeightBytes)
    return fail(CONVROT_ERR_UNSUPPORTED, "blocked activations are limited to 2 GiB (M=%lld K=%lld)", (long long)M,
                (long long)K);
  if (packed_weight_bytes(N, K) >= kMaxWeightBytes)
    return fail(CONVROT_ERR_UNSUPPORTED, "W4A4 GEMM packed weights are limited to 2 GiB (N=%lld K=%lld)", (long long)N,
                (long long)K);
  if (M == 0 || N == 0) return ok();
  if (!act || !xscales || !qweight || !wscales || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(act, 16) || !aligned(qweight, 16) || !aligned(out, 16))
    return fail(CONVROT_ERR_INVALID, "act, qweight and out must be 16-byte aligned");
  return ok();
}

}  // namespace

int convrot_w4a4_gemm(const void* act, int act_format, const float* xscales, const uint8_t* qweight,
                      const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K, void* out,
                      int out_dtype, void* stream) {
  if (int rc = check_w4a4(act, act_format, xscales, qweight, wscales, M, N, K, out, out_dtype)) return rc;
  if (M == 0 || N == 0) return ok();
  return launch_status(convrot::launch_w4a4_gemm(act, act_format, xscales, qweight, wscales, bias, M, N, K, out,
                                                 out_dtype, (hipStream_t)stream),
                       "convrot_w4a4_gemm");
}

namespace {

int check_fp6(const uint8_t* act6, const float* xscales, const uint8_t* w6, const float* wscales, int64_t M,
              int64_t N, int64_t K, void* out, int out_dtype, int* odt) {
  if (M < 0 || N < 0 || K <= 0 || K % 128 || M > INT32_MAX || N > INT32_MAX || K >= 262144)
    return fail(CONVROT_ERR_INVALID,
                "FP6 W4A4 GEMM: bad shape M=%lld N=%lld K=%lld (K a multiple of 128 below 262144)", (long long)M,
                (long long)N, (long long)K);
  if (convrot_fp6_bytes(M, K) > kMaxFp6OperandBytes || convrot_fp6_bytes(N, K) > kMaxFp6OperandBytes)
    return fail(CONVROT_ERR_UNSUPPORTED,
                "FP6 W4A4 GEMM: an operand of M=%lld or N=%lld rows at K=%lld exceeds %lld FP6 bytes (32-bit "
                "buffer offsets); use the INT8 GEMM",
                (long long)M, (long long)N, (long long)K, (long long)kMaxFp6OperandBytes);
  if (out_dtype != CONVROT_DTYPE_BF16 && out_dtype != CONVROT_DTYPE_F16 && out_dtype != CONVROT_DTYPE_F32)
    return fail(CONVROT_ERR_INVALID, "unsupported output dtype %d", out_dtype);
  *odt = out_dtype == CONVROT_DTYPE_BF16 ? convrot::kBF16 : out_dtype == CONVROT_DTYPE_F16 ? convrot::kF16
                                                                                             : convrot::kF32;
  if (M == 0 || N == 0) return ok();
  if (!act6 || !xscales || !w6 || !wscales || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(act6, 16) || !aligned(w6, 16) || !aligned(out, 16))
    return fail(CONVROT_ERR_INVALID, "act6, w6 and out must be 16-byte aligned");
  return ok();
}

}  // namespace

int convrot_w4a4_gemm_fp6(const uint8_t* act6, const float* xscales, const uint8_t* w6, const float* wscales,
                          const float* bias, int64_t M, int64_t N, int64_t K, void* out, int out_dtype, void* stream) {
  int odt = 0;
  if (int rc = check_fp6(act6, xscales, w6, wscales, M, N, K, out, out_dtype, &odt)) return rc;
  if (M == 0 || N == 0) return ok();
  return launch_status(convrot::launch_w4a4_gemm_fp6(act6, xscales, w6, wscales, bias, M, N, K, out, odt,
                                                     (hipStream_t)stream, convrot::GatedResidual{}),
                       "convrot_w4a4_gemm_fp6");
}

namespace {

// Checks of the gated-residual arguments shared by both GEMMs (after the GEMM's
// own checks, with M, N > 0); fills `gr` on success.
int check_residual(const void* residual, const void* gate, int64_t gate_stride, int64_t rows_per_gate, int64_t M,
                   int64_t N, convrot::GatedResidual* gr) {
  if (!residual) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(residual, 16) || (gate && !aligned(gate, 16)))
    return fail(CONVROT_ERR_INVALID, "residual and gate must be 16-byte aligned");
  // Any rows_per_gate >= M selects gate row 0 for every output row.
  const int64_t rpg = gate ? (rows_per_gate < M ? rows_per_gate : M) : 1;
  if (gate && (M + rpg - 1) / rpg > 1 && gate_stride < N)
    return fail(CONVROT_ERR_INVALID, "gate rows %lld elements apart overlap (N=%lld)", (long long)gate_stride,
                (long long)N);
  *gr = convrot::GatedResidual{residual, gate, gate ? gate_stride : 0, (int)rpg};
  return ok();
}

}  // namespace

int convrot_w4a4_gemm_residual(const void* act, int act_format, const float* xscales, const uint8_t* qweight,
                               const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K,
                               const void* residual, const void* gate, int64_t gate_stride,
                               int64_t rows_per_gate, void* out, int out_dtype, void* stream) {
  if (int rc = check_w4a4(act, act_format, xscales, qweight, wscales, M, N, K, out, out_dtype)) return rc;
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (M == 0 || N == 0) return ok();
  convrot::GatedResidual gr{};
  if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  return launch_status(convrot::launch_w4a4_gemm(act, act_format, xscales, qweight, wscales, bias, M, N, K, out,
                                                 out_dtype, (hipStream_t)stream, gr),
                       "convrot_w4a4_gemm_residual");
}

int convrot_w4a4_gemm_fp6_residual(const uint8_t* act6, const float* xscales, const uint8_t* w6,
                                   const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K,
                                   const void* residual, const void* gate, int64_t gate_stride,
                                   int64_t rows_per_gate, void* out, int out_dtype, void* stream) {
  int odt = 0;
  if (int rc = check_fp6(act6, xscales, w6, wscales, M, N, K, out, out_dtype, &odt)) return rc;
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (M == 0 || N == 0) return ok();
  convrot::GatedResidual gr{};
  if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  return launch_status(convrot::launch_w4a4_gemm_fp6(act6, xscales, w6, wscales, bias, M, N, K, out, odt,
                                                     (hipStream_t)stream, gr),
                       "convrot_w4a4_gemm_fp6_residual");
}

int convrot_w4a4_gemm_fp6_compact(const uint8_t* act6, const float* xscales, const uint8_t* w6c,
                                  const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K,
                                  const void* residual, const void* gate, int64_t gate_stride,
                                  int64_t rows_per_gate, void* out, int out_dtype, void* stream) {
  int odt = 0;
  if (int rc = check_fp6(act6, xscales, w6c, wscales, M, N, K, out, out_dtype, &odt)) return rc;
  if (gate && !residual) return fail(CONVROT_ERR_INVALID, "a gate needs a residual");
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (M == 0 || N == 0) return ok();
  convrot::GatedResidual gr{};
  if (residual)
    if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  return launch_status(convrot::launch_w4a4_gemm_fp6(act6, xscales, w6c, wscales, bias, M, N, K, out, odt,
                                                     (hipStream_t)stream, gr, true),
                       "convrot_w4a4_gemm_fp6_compact");
}

int64_t convrot_w4a4_workspace_bytes(void) { return (int64_t)convrot::kSkWorkspaceBytes; }

int convrot_w4a4_gemm_ws(const void* act, int act_format, const float* xscales, const uint8_t* qweight,
                         const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K,
                         const void* residual, const void* gate, int64_t gate_stride, int64_t rows_per_gate,
                         void* workspace, int64_t workspace_bytes, void* out, int out_dtype, void* stream) {
  if (int rc = check_w4a4(act, act_format, xscales, qweight, wscales, M, N, K, out, out_dtype)) return rc;
  if (workspace_bytes < 0 || (workspace_bytes > 0 && !workspace))
    return fail(CONVROT_ERR_INVALID, "invalid workspace (%lld bytes)", (long long)workspace_bytes);
  if (workspace && !aligned(workspace, 256)) return fail(CONVROT_ERR_INVALID, "workspace must be 256-byte aligned");
  if (gate && !residual) return fail(CONVROT_ERR_INVALID, "a gate needs a residual");
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (M == 0 || N == 0) return ok();
  convrot::GatedResidual gr{};
  if (residual)
    if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  convrot::WorkspaceSource src;
  src.kind = convrot::WorkspaceSource::kGiven;
  src.given = {(uint8_t*)workspace, workspace ? (size_t)workspace_bytes : 0};
  return launch_status(convrot::launch_w4a4_gemm(act, act_format, xscales, qweight, wscales, bias, M, N, K, out,
                                                 out_dtype, (hipStream_t)stream, gr, src),
                       "convrot_w4a4_gemm_ws");
}

int convrot_w4a4_gemm_noalloc(const void* act, int act_format, const float* xscales, const uint8_t* qweight,
                              const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K,
                              const void* residual, const void* gate, int64_t gate_stride, int64_t rows_per_gate,
                              void* out, int out_dtype, void* stream) {
  if (int rc = check_w4a4(act, act_format, xscales, qweight, wscales, M, N, K, out, out_dtype)) return rc;
  if (gate && !residual) return fail(CONVROT_ERR_INVALID, "a gate needs a residual");
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (M == 0 || N == 0) return ok();
  convrot::GatedResidual gr{};
  if (residual)
    if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  // The plan of convrot_w4a4_gemm_ws with a full workspace; its workspace must fit the static scratch.
  const size_t need = convrot::w4a4_plan_workspace_bytes(act_format, M, N, K);
  if (need > convrot::kNoAllocScratchBytes)
    return fail(CONVROT_ERR_INVALID,
                "convrot_w4a4_gemm_noalloc: the plan for M=%lld N=%lld K=%lld needs %zu bytes of scratch, beyond "
                "the static maximum of %zu",
                (long long)M, (long long)N, (long long)K, need, convrot::kNoAllocScratchBytes);
  convrot::WorkspaceSource src;
  src.kind = convrot::WorkspaceSource::kGiven;
  if (need > 0) {
    if (const hipError_t e = convrot::noalloc_scratch((hipStream_t)stream, &src.given); e != hipSuccess)
      return fail(CONVROT_ERR_LAUNCH, "convrot_w4a4_gemm_noalloc: scratch set-up failed: %s", hipGetErrorString(e));
  }
  return launch_status(convrot::launch_w4a4_gemm(act, act_format, xscales, qweight, wscales, bias, M, N, K, out,
                                                 out_dtype, (hipStream_t)stream, gr, src),
                       "convrot_w4a4_gemm_noalloc");
}

int convrot_w4a4_status(const void* workspace, void* stream) {
  const char* what = nullptr;
  const int rc = convrot::w4a4_workspace_status(workspace, (hipStream_t)stream, &what);
  if (rc < 0) return fail(CONVROT_ERR_LAUNCH, "convrot_w4a4_status: %s", hipGetErrorString(hipGetLastError()));
  if (rc > 0) return fail(CONVROT_ERR_LAUNCH, "%s", what);
  return ok();
}

namespace {

// Argument checks of the W4A16 GEMM entry points; CONVROT_OK when the launch
// may proceed (M == 0 or N == 0 included).
int check_w4a16(const void* act, int act_dtype, const uint8_t* qweight, const float* wscales, int64_t M, int64_t N,
                int64_t K, void* out, int out_dtype) {
  if (act_dtype != CONVROT_DTYPE_F16 && act_dtype != CONVROT_DTYPE_BF16)
    return fail(CONVROT_ERR_INVALID, "MPP W4A16 requires float16 or bfloat16 activation, got %s", dtype_name(act_dtype));
  if (!valid_dtype(out_dtype)) return fail(CONVROT_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 0 || K <= 0) return fail(CONVROT_ERR_INVALID, "invalid GEMM shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (K % 32) return fail(CONVROT_ERR_INVALID, "W4A16 GEMM requires K divisible by 32, got %lld", (long long)K);
  if (K > kMaxFeatures)
    return fail(CONVROT_ERR_UNSUPPORTED, "W4A16 GEMM supports K up to %lld, got %lld", (long long)kMaxFeatures, (long long)K);
  if (M > 0x7fffffff || N > 0x7fffffff) return fail(CONVROT_ERR_UNSUPPORTED, "GEMM dimension too large");
  if (packed_weight_bytes(N, K) >= kMaxWeightBytes)
    return fail(CONVROT_ERR_UNSUPPORTED, "W4A16 GEMM packed weights are limited to 2 GiB (N=%lld K=%lld)", (long long)N,
                (long long)K);
  if (M == 0 || N == 0) return ok();
  if (!act || !qweight || !wscales || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(act, 16) || !aligned(qweight, 16) || !aligned(out, 16))
    return fail(CONVROT_ERR_INVALID, "act, qweight and out must be 16-byte aligned");
  return ok();
}

}  // namespace

int convrot_w4a16_gemm(const void* act, int act_dtype, const uint8_t* qweight, const float* wscales,
                       const float* bias, int64_t M, int64_t N, int64_t K, void* out, int out_dtype, void* stream) {
  if (int rc = check_w4a16(act, act_dtype, qweight, wscales, M, N, K, out, out_dtype)) return rc;
  if (M == 0 || N == 0) return ok();
  return launch_status(convrot::launch_w4a16_gemm(act, act_dtype, qweight, wscales, bias, M, N, K, out, out_dtype,
                                                  (hipStream_t)stream),
                       "convrot_w4a16_gemm");
}

int convrot_w4a16_gemm_residual(const void* act, int act_dtype, const uint8_t* qweight, const float* wscales,
                                const float* bias, int64_t M, int64_t N, int64_t K, const void* residual,
                                const void* gate, int64_t gate_stride, int64_t rows_per_gate, void* out,
                                int out_dtype, void* stream) {
  if (int rc = check_w4a16(act, act_dtype, qweight, wscales, M, N, K, out, out_dtype)) return rc;
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (M == 0 || N == 0) return ok();
  convrot::GatedResidual gr{};
  if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  return launch_status(convrot::launch_w4a16_gemm(act, act_dtype, qweight, wscales, bias, M, N, K, out, out_dtype,
                                                  (hipStream_t)stream, gr),
                       "convrot_w4a16_gemm_residual");
}

int convrot_w4a16_gemm_ws(const void* act, int act_dtype, const uint8_t* qweight, const float* wscales,
                          const float* bias, int64_t M, int64_t N, int64_t K, const void* residual, const void* gate,
                          int64_t gate_stride, int64_t rows_per_gate, void* workspace, int64_t workspace_bytes,
                          void* out, int out_dtype, void* stream) {
  if (int rc = check_w4a16(act, act_dtype, qweight, wscales, M, N, K, out, out_dtype)) return rc;
  if (workspace_bytes < 0 || (workspace_bytes > 0 && !workspace))
    return fail(CONVROT_ERR_INVALID, "invalid workspace (%lld bytes)", (long long)workspace_bytes);
  if (workspace && !aligned(workspace, 256)) return fail(CONVROT_ERR_INVALID, "workspace must be 256-byte aligned");
  if (gate && !residual) return fail(CONVROT_ERR_INVALID, "a gate needs a residual");
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (M == 0 || N == 0) return ok();
  convrot::GatedResidual gr{};
  if (residual)
    if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  const convrot::Workspace work{(uint8_t*)workspace, workspace ? (size_t)workspace_bytes : 0};
  return launch_status(convrot::launch_w4a16_gemm(act, act_dtype, qweight, wscales, bias, M, N, K, out, out_dtype,
                                                  (hipStream_t)stream, gr, work),
                       "convrot_w4a16_gemm_ws");
}

int convrot_linear_rows(const void* x, int dtype, int group_size, int a4, const uint8_t* qweight,
                        const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K,
                        const void* residual, const void* gate, int64_t gate_stride, int64_t rows_per_gate, void* out,
                        void* stream) {
  if (!valid_dtype(dtype)) return fail(CONVROT_ERR_INVALID, "unsupported activation dtype code %d", dtype);
  if (M < 0 || N < 0 || K <= 0)
    return fail(CONVROT_ERR_INVALID, "invalid shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  const int s = log4_group(group_size);
  if (s < 0) return fail(CONVROT_ERR_INVALID, "Regular Hadamard size must be a power of 4, got %d", group_size);
  if (K % group_size)
    return fail(CONVROT_ERR_INVALID, "features %lld not divisible by ConvRot group size %d", (long long)K, group_size);
  if (N > 0x7fffffff || packed_weight_bytes(N, K) >= kMaxWeightBytes)
    return fail(CONVROT_ERR_UNSUPPORTED, "packed weights are limited to 2 GiB (N=%lld K=%lld)", (long long)N,
                (long long)K);
  if (gate && !residual) return fail(CONVROT_ERR_INVALID, "a gate needs a residual");
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (M == 0 || N == 0) return ok();
  if (!convrot::linear_rows_eligible(M, K, dtype, s, a4 != 0))
    return fail(CONVROT_ERR_UNSUPPORTED,
                "the few-row linear takes 1 to 16 rows of at most 32 KB in all, groups of 64 or 256 and (W4A16) "
                "16-bit activations; got M=%lld K=%lld group %d %s",
                (long long)M, (long long)K, group_size, dtype_name(dtype));
  if (!x || !qweight || !wscales || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(x, 16) || !aligned(qweight, 16) || !aligned(out, 16))
    return fail(CONVROT_ERR_INVALID, "x, qweight and out must be 16-byte aligned");
  // every workgroup reads all of x, so no workgroup may write into it
  const int64_t esize = dtype == CONVROT_DTYPE_F32 ? 4 : 2;
  const uintptr_t xa = (uintptr_t)x, oa = (uintptr_t)out;
  if (xa < oa + (uintptr_t)(M * N * esize) && oa < xa + (uintptr_t)(M * K * esize))
    return fail(CONVROT_ERR_INVALID, "out must not overlap x");
  convrot::GatedResidual gr{};
  if (residual)
    if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  return launch_status(convrot::launch_linear_rows(x, dtype, s, a4 != 0, qweight, wscales, bias, M, N, K, out, gr,
                                                   (hipStream_t)stream),
                       "convrot_linear_rows");
}

int convrot_pack_int4(const int8_t* values, int64_t rows, int64_t packed_cols, uint8_t* out, void* stream) {
  if (rows < 0 || packed_cols < 0) return fail(CONVROT_ERR_INVALID, "invalid pack shape");
  if (rows * packed_cols == 0) return ok();
  if (!values || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(values, 2)) return fail(CONVROT_ERR_INVALID, "values must be 2-byte aligned");
  return launch_status(convrot::launch_pack_int4(values, rows, packed_cols, out, (hipStream_t)stream),
                       "convrot_pack_int4");
}

int convrot_unpack_int4(const uint8_t* packed, int64_t rows, int64_t packed_cols, int8_t* out, void* stream) {
  if (rows < 0 || packed_cols < 0) return fail(CONVROT_ERR_INVALID, "invalid unpack shape");
  if (rows * packed_cols == 0) return ok();
  if (!packed || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(out, 2)) return fail(CONVROT_ERR_INVALID, "out must be 2-byte aligned");
  return launch_status(convrot::launch_unpack_int4(packed, rows, packed_cols, out, (hipStream_t)stream),
                       "convrot_unpack_int4");
}

int convrot_repack_weight(const uint8_t* in, int in_layout, uint8_t* out, int out_layout, int64_t N, int64_t K,
                          void* stream) {
  auto valid_layout = [](int l) {
    return l == CONVROT_LAYOUT_NK || l == CONVROT_LAYOUT_KN || l == CONVROT_LAYOUT_CDNA4;
  };
  if (!valid_layout(in_layout) || !valid_layout(out_layout))
    return fail(CONVROT_ERR_INVALID, "unknown weight layout %d -> %d", in_layout, out_layout);
  if (N < 0 || K < 0) return fail(CONVROT_ERR_INVALID, "invalid weight shape (%lld, %lld)", (long long)N, (long long)K);
  if ((in_layout == CONVROT_LAYOUT_KN || out_layout == CONVROT_LAYOUT_KN) && (N % 2))
    return fail(CONVROT_ERR_INVALID, "MPP int4 packing requires even out_features, got %lld", (long long)N);
  if ((in_layout == CONVROT_LAYOUT_NK || out_layout == CONVROT_LAYOUT_NK) && (K % 2))
    return fail(CONVROT_ERR_INVALID, "row-major int4 packing requires even in_features, got %lld", (long long)K);
  if (N == 0 || K == 0) return ok();
  if (!in || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (in == out) return fail(CONVROT_ERR_INVALID, "repack cannot run in place");
  return launch_status(convrot::launch_repack(in, in_layout, out, out_layout, N, K, (hipStream_t)stream),
                       "convrot_repack_weight");
}

int convrot_weight_fp6_compact(const uint8_t* cdna4, uint8_t* fp6c, int* minus8, int64_t N, int64_t K,
                               void* stream) {
  if (N < 0 || K < 0) return fail(CONVROT_ERR_INVALID, "invalid weight shape (%lld, %lld)", (long long)N, (long long)K);
  if (K % 128)
    return fail(CONVROT_ERR_UNSUPPORTED, "FP6 operands require in_features divisible by 128, got %lld",
                (long long)K);
  if ((N == 0 || K == 0) && !minus8) return ok();
  if (((N && K) && (!cdna4 || !fp6c))) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(cdna4, 16) || !aligned(fp6c, 16) || !aligned(minus8, 4))
    return fail(CONVROT_ERR_INVALID, "cdna4 and fp6c must be 16-byte aligned, minus8 4-byte aligned");
  return launch_status(convrot::launch_weight_fp6c(cdna4, fp6c, minus8, N, K, (hipStream_t)stream),
                       "convrot_weight_fp6_compact");
}

int convrot_weight_fp6(const uint8_t* cdna4, uint8_t* fp6, int64_t N, int64_t K, void* stream) {
  if (N < 0 || K < 0) return fail(CONVROT_ERR_INVALID, "invalid weight shape (%lld, %lld)", (long long)N, (long long)K);
  if (K % 128)
    return fail(CONVROT_ERR_UNSUPPORTED, "FP6 operands require in_features divisible by 128, got %lld",
                (long long)K);
  if (N == 0 || K == 0) return ok();
  if (!cdna4 || !fp6) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(cdna4, 16) || !aligned(fp6, 16)) return fail(CONVROT_ERR_INVALID, "cdna4 and fp6 must be 16-byte aligned");
  return launch_status(convrot::launch_weight_fp6(cdna4, fp6, N, K, (hipStream_t)stream),
                       "convrot_weight_fp6");
}

namespace {

constexpr int64_t kMaxInt8Stride = int64_t(1) << 22;  // of a W8A8 operand's rows: a tile's offsets stay below 2^31
constexpr int64_t kMaxRows = 0x7fffffff;

// Checks shared by the row operators; `features` may not exceed `most`.
int check_rows(const char* what, const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride,
               int64_t most) {
  if (!valid_dtype(dtype)) return fail(CONVROT_ERR_INVALID, "unsupported activation dtype code %d", dtype);
  if (rows < 0 || features < 0)
    return fail(CONVROT_ERR_INVALID, "invalid shape rows=%lld features=%lld", (long long)rows, (long long)features);
  if (features > most)
    return fail(CONVROT_ERR_UNSUPPORTED, "%s supports at most %lld features, got %lld", what, (long long)most,
                (long long)features);
  if (rows > kMaxRows) return fail(CONVROT_ERR_UNSUPPORTED, "%s supports at most 2^31-1 rows", what);
  if (rows == 0 || features == 0) return ok();
  if (!x) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (rows > 1 && x_stride < 0) return fail(CONVROT_ERR_INVALID, "negative row stride %lld", (long long)x_stride);
  if (!aligned(x, dtype == CONVROT_DTYPE_F32 ? 4 : 2)) return fail(CONVROT_ERR_INVALID, "x is not aligned to its type");
  return ok();
}

int check_codes(const int8_t* codes, int64_t stride, int64_t features, const float* scales) {
  if (!codes || !scales) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (stride < features || stride % 16 || !aligned(codes, 16))
    return fail(CONVROT_ERR_INVALID, "codes need 16-byte aligned rows of at least %lld bytes, got a stride of %lld",
                (long long)features, (long long)stride);
  if (stride > (features + 15) / 16 * 16 + 1024 || stride > 65536)
    return fail(CONVROT_ERR_UNSUPPORTED, "codes stride %lld too long for %lld features", (long long)stride,
                (long long)features);
  return ok();
}

int check_params(const void* gain, const void* shift, int dtype, int param_dtype, int64_t rows,
                 int64_t rows_per_vector) {
  if (!gain && !shift && rows_per_vector <= 0) return ok();
  if (param_dtype != dtype && param_dtype != CONVROT_DTYPE_F32)
    return fail(CONVROT_ERR_INVALID, "norm parameters must have the activations' type or float32, got %s",
                dtype_name(param_dtype));
  if (rows_per_vector <= 0 || rows % rows_per_vector)
    return fail(CONVROT_ERR_INVALID, "%lld rows do not split into vectors of %lld rows", (long long)rows,
                (long long)rows_per_vector);
  const uintptr_t a = param_dtype == CONVROT_DTYPE_F32 ? 4 : 2;
  if (!aligned(gain, a) || !aligned(shift, a))
    return fail(CONVROT_ERR_INVALID, "norm parameters are not aligned to their type");
  return ok();
}

int check_rotary(int dtype, int batch, int q_heads, int k_heads, int64_t length, int dim, const float* table,
                 int pairs, int64_t table_batch_stride, const void* q_weight, const void* k_weight, int weight_dtype,
                 const int64_t* strides) {
  if (!valid_dtype(dtype)) return fail(CONVROT_ERR_INVALID, "unsupported activation dtype code %d", dtype);
  if (batch < 0 || q_heads < 0 || k_heads < 0 || length < 0 || dim < 0 || pairs < 0)
    return fail(CONVROT_ERR_INVALID, "invalid rotary shape batch=%d heads=%d/%d length=%lld dim=%d pairs=%d", batch,
                q_heads, k_heads, (long long)length, dim, pairs);
  if (2 * (int64_t)pairs > dim)
    return fail(CONVROT_ERR_INVALID, "%d pairs do not fit a head of %d features", pairs, dim);
  if (dim > 512) return fail(CONVROT_ERR_UNSUPPORTED, "rotary positions support heads of up to 512 features, got %d", dim);
  if (q_heads > 65536 || k_heads > 65536 || (int64_t)batch * length > kMaxRows || length > kMaxRows)
    return fail(CONVROT_ERR_UNSUPPORTED, "rotary positions support at most 2^31-1 tokens and 65536 heads");
  if ((q_weight || k_weight) && weight_dtype != dtype && weight_dtype != CONVROT_DTYPE_F32)
    return fail(CONVROT_ERR_INVALID, "norm weights must have the activations' type or float32, got %s",
                dtype_name(weight_dtype));
  if (batch == 0 || length == 0 || dim == 0 || q_heads + k_heads == 0) return ok();
  if (!strides || (pairs > 0 && !table)) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(table, 4) || table_batch_stride < 0) return fail(CONVROT_ERR_INVALID, "invalid rotary table");
  return ok();
}

}  // namespace

int convrot_quantize_int8(const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride, int8_t* codes,
                          int64_t codes_stride, float* scales, void* stream) {
  if (int rc = check_rows("8-bit quantization", x, dtype, rows, features, x_stride, kMaxFeatures)) return rc;
  if (rows == 0 || features == 0) return ok();
  if (int rc = check_codes(codes, codes_stride, features, scales)) return rc;
  return launch_status(convrot::launch_quantize_int8(x, dtype, rows, features, x_stride, codes, codes_stride, scales,
                                                     (hipStream_t)stream),
                       "convrot_quantize_int8");
}

namespace {

// Checks of a W8A8 product but for its activations; CONVROT_OK when the launch
// may proceed (M == 0 or N == 0 included).
int check_w8a8(int64_t M, int64_t N, int64_t K, const int8_t* weight, int64_t weight_stride, const float* wscales,
               const void* gate, const void* residual, int64_t rows_per_gate, const void* workspace,
               int64_t workspace_bytes, const void* out, int out_dtype) {
  if (!valid_dtype(out_dtype)) return fail(CONVROT_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 0 || K <= 0)
    return fail(CONVROT_ERR_INVALID, "invalid GEMM shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (K > kMaxFeatures)
    return fail(CONVROT_ERR_UNSUPPORTED, "W8A8 GEMM supports K up to %lld, got %lld", (long long)kMaxFeatures, (long long)K);
  // 2^31 - 1 less what rounding a dimension up to whole tiles adds
  if (M > 0x7ffffe00 || N > 0x7ffffe00) return fail(CONVROT_ERR_UNSUPPORTED, "GEMM dimension too large");
  if (gate && !residual) return fail(CONVROT_ERR_INVALID, "a gate needs a residual");
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (workspace_bytes < 0 || (workspace_bytes > 0 && !workspace))
    return fail(CONVROT_ERR_INVALID, "invalid workspace (%lld bytes)", (long long)workspace_bytes);
  if (workspace && !aligned(workspace, 256)) return fail(CONVROT_ERR_INVALID, "workspace must be 256-byte aligned");
  if (M == 0 || N == 0) return ok();
  if (!weight || !wscales || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (weight_stride < (K + 15) / 16 * 16 || weight_stride % 16 || !aligned(weight, 16) || !aligned(out, 16))
    return fail(CONVROT_ERR_INVALID,
                "W8A8 operands need 16-byte aligned rows that cover K rounded up to 16 (K=%lld, weight stride %lld)",
                (long long)K, (long long)weight_stride);
  if (weight_stride > kMaxInt8Stride)
    return fail(CONVROT_ERR_UNSUPPORTED, "W8A8 row strides are limited to %lld bytes", (long long)kMaxInt8Stride);
  return ok();
}

}  // namespace

int convrot_w8a8_gemm(const int8_t* act, int64_t act_stride, const float* xscales, const int8_t* weight,
                      int64_t weight_stride, const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K,
                      const void* residual, const void* gate, int64_t gate_stride, int64_t rows_per_gate,
                      void* workspace, int64_t workspace_bytes, void* out, int out_dtype, void* stream) {
  if (int rc = check_w8a8(M, N, K, weight, weight_stride, wscales, gate, residual, rows_per_gate, workspace,
                          workspace_bytes, out, out_dtype))
    return rc;
  if (M == 0 || N == 0) return ok();
  if (!act || !xscales) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (act_stride < (K + 15) / 16 * 16 || act_stride % 16 || !aligned(act, 16))
    return fail(CONVROT_ERR_INVALID,
                "W8A8 operands need 16-byte aligned rows that cover K rounded up to 16 (K=%lld, activation stride %lld)",
                (long long)K, (long long)act_stride);
  if (act_stride > kMaxInt8Stride)
    return fail(CONVROT_ERR_UNSUPPORTED, "W8A8 row strides are limited to %lld bytes", (long long)kMaxInt8Stride);
  convrot::GatedResidual gr{};
  if (residual)
    if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  const convrot::Workspace work{(uint8_t*)workspace, workspace ? (size_t)workspace_bytes : 0};
  return launch_status(convrot::launch_w8a8_gemm(act, act_stride, xscales, weight, weight_stride, wscales, bias, M, N,
                                                 K, out, out_dtype, (hipStream_t)stream, gr, work),
                       "convrot_w8a8_gemm");
}

int64_t convrot_w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > kMaxFeatures || M > 0x7ffffe00 || N > 0x7ffffe00) return 0;
  return convrot::w8a8_workspace_bytes(M, N, K);
}

// Rows of codes in whole cache lines (rows of 2112 bytes: the product 10 % slower).
static int64_t codes_stride_of(int64_t K) { return (K + 127) / 128 * 128; }

int64_t convrot_w8a8_scratch_bytes(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0) return 0;
  return M * codes_stride_of(K) + M * 4;
}

int convrot_w8a8_linear(const void* x, int dtype, int64_t x_stride, const int8_t* weight, int64_t weight_stride,
                        const float* wscales, const float* bias, int64_t M, int64_t N, int64_t K,
                        const void* residual, const void* gate, int64_t gate_stride, int64_t rows_per_gate,
                        void* scratch, int64_t scratch_bytes, void* workspace, int64_t workspace_bytes, void* out,
                        void* stream) {
  if (int rc = check_rows("8-bit quantization", x, dtype, M, K, x_stride, kMaxFeatures)) return rc;
  if (int rc = check_w8a8(M, N, K, weight, weight_stride, wscales, gate, residual, rows_per_gate, workspace,
                          workspace_bytes, out, dtype))
    return rc;
  if (M == 0 || N == 0) return ok();
  convrot::GatedResidual gr{};
  if (residual)
    if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  const convrot::Workspace work{(uint8_t*)workspace, workspace ? (size_t)workspace_bytes : 0};
  // a fused launch's workgroups all read x: none may write into it
  const int64_t es = dtype == CONVROT_DTYPE_F32 ? 4 : 2;
  const uintptr_t xa = (uintptr_t)x, oa = (uintptr_t)out;
  const bool apart = oa + (uintptr_t)(M * N * es) <= xa || xa + (uintptr_t)(((M - 1) * x_stride + K) * es) <= oa;
  if (apart && convrot::w8a8_fused(x, dtype, M, K, x_stride))
    return launch_status(convrot::launch_w8a8_fused(x, x_stride, dtype, weight, weight_stride, wscales, bias, M, N, K,
                                                    out, (hipStream_t)stream, gr, work),
                         "convrot_w8a8_linear");
  const int64_t need = convrot_w8a8_scratch_bytes(M, K);
  convrot::Workspace rest = work;
  if (!scratch && need <= workspace_bytes / 4) {
    // the end of the workspace, away from the partial sums that share K and never over the control
    // block in front of them, whose words stay zero between launches
    const size_t left = (size_t)(workspace_bytes - need) & ~(size_t)255;
    if (left >= convrot::kW8a8PartialOffset) {
      rest.bytes = left;
      scratch = rest.ptr + left;
      scratch_bytes = need;
    }
  }
  if (!scratch || !aligned(scratch, 16) || scratch_bytes < need)
    return fail(CONVROT_ERR_INVALID, "the W8A8 linear needs a 16-byte aligned scratch buffer of %lld bytes, got %lld",
                (long long)need, (long long)scratch_bytes);
  const int64_t stride = codes_stride_of(K);
  int8_t* codes = (int8_t*)scratch;
  float* scales = (float*)(codes + M * stride);
  hipError_t e = convrot::launch_quantize_int8(x, dtype, M, K, x_stride, codes, stride, scales, (hipStream_t)stream);
  if (e == hipSuccess)
    e = convrot::launch_w8a8_gemm(codes, stride, scales, weight, weight_stride, wscales, bias, M, N, K, out, dtype,
                                  (hipStream_t)stream, gr, rest);
  return launch_status(e, "convrot_w8a8_linear");
}

int convrot_w8a8_fused(const void* x, int dtype, int64_t M, int64_t K, int64_t x_stride) {
  return M > 0 && K > 0 && valid_dtype(dtype) && convrot::w8a8_fused(x, dtype, M, K, x_stride) ? 1 : 0;
}

int convrot_layer_norm(const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride, const void* gain,
                       const void* shift, int param_dtype, int plus_one, int64_t rows_per_vector, float eps,
                       void* out, float* mean, float* rstd, void* stream) {
  if (int rc = check_rows("layer norm", x, dtype, rows, features, x_stride, kMaxFeatures)) return rc;
  if (int rc = check_params(gain, shift, dtype, param_dtype, rows, rows_per_vector)) return rc;
  if (!mean != !rstd) return fail(CONVROT_ERR_INVALID, "mean and rstd come together");
  if (rows == 0 || features == 0) return ok();
  if (!out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(out, dtype == CONVROT_DTYPE_F32 ? 4 : 2)) return fail(CONVROT_ERR_INVALID, "out is not aligned to its type");
  return launch_status(convrot::launch_layer_norm(x, dtype, rows, features, x_stride, gain, shift, param_dtype,
                                                  plus_one != 0, rows_per_vector, eps, out, mean, rstd,
                                                  (hipStream_t)stream),
                       "convrot_layer_norm");
}

int convrot_layer_norm_int8(const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride,
                            const void* gain, const void* shift, int param_dtype, int plus_one,
                            int64_t rows_per_vector, float eps, int8_t* codes, int64_t codes_stride, float* scales,
                            void* stream) {
  if (int rc = check_rows("layer norm", x, dtype, rows, features, x_stride, kMaxFeatures)) return rc;
  if (int rc = check_params(gain, shift, dtype, param_dtype, rows, rows_per_vector)) return rc;
  if (rows == 0 || features == 0) return ok();
  if (int rc = check_codes(codes, codes_stride, features, scales)) return rc;
  return launch_status(convrot::launch_layer_norm_int8(x, dtype, rows, features, x_stride, gain, shift, param_dtype,
                                                       plus_one != 0, rows_per_vector, eps, codes, codes_stride,
                                                       scales, (hipStream_t)stream),
                       "convrot_layer_norm_int8");
}

int64_t convrot_layer_norm_workspace_bytes(int64_t rows, int64_t features, int64_t rows_per_vector) {
  if (rows <= 0 || features <= 0 || rows_per_vector <= 0 || rows % rows_per_vector) return 0;
  return (rows / rows_per_vector) * convrot::layer_norm_parts(rows, features, rows_per_vector) * 2 * features * 4;
}

int convrot_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* mean,
                                const float* rstd, int dtype, int64_t rows, int64_t features, const void* gain,
                                int param_dtype, int plus_one, int64_t rows_per_vector, void* dx, void* dgain,
                                void* dshift, void* workspace, int64_t workspace_bytes, void* stream) {
  constexpr int64_t most = 32768;  // a thread keeps the gradient sums of 32 features
  if (int rc = check_rows("the layer norm's gradient", x, dtype, rows, features, x_stride, most)) return rc;
  if (int rc = check_rows("the layer norm's gradient", dy, dtype, rows, features, dy_stride, most)) return rc;
  if (rows_per_vector <= 0) return fail(CONVROT_ERR_INVALID, "rows_per_vector must be positive, got %lld", (long long)rows_per_vector);
  if (int rc = check_params(gain, nullptr, dtype, param_dtype, rows, rows_per_vector)) return rc;
  if (rows == 0 || features == 0) return ok();
  if (!mean || !rstd || !dx) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(dx, dtype == CONVROT_DTYPE_F32 ? 4 : 2)) return fail(CONVROT_ERR_INVALID, "dx is not aligned to its type");
  if ((dgain || dshift) &&
      (!workspace || !aligned(workspace, 16) ||
       workspace_bytes < convrot_layer_norm_workspace_bytes(rows, features, rows_per_vector)))
    return fail(CONVROT_ERR_INVALID, "the layer norm's gradient needs a 16-byte aligned workspace of %lld bytes, got %lld",
                (long long)convrot_layer_norm_workspace_bytes(rows, features, rows_per_vector),
                (long long)workspace_bytes);
  return launch_status(convrot::launch_layer_norm_backward(dy, dy_stride, x, x_stride, mean, rstd, dtype, rows,
                                                           features, gain, param_dtype, plus_one != 0,
                                                           rows_per_vector, dx, dgain, dshift, (float*)workspace,
                                                           (hipStream_t)stream),
                       "convrot_layer_norm_backward");
}

int convrot_axes_table(const void* positions, int kind, int64_t rows, int axes, const int* dims, double theta,
                       float* out, void* stream) {
  if (kind < CONVROT_POS_F32 || kind > CONVROT_POS_I64) return fail(CONVROT_ERR_INVALID, "unknown position type %d", kind);
  if (axes < 1 || axes > 8 || !dims) return fail(CONVROT_ERR_INVALID, "positions need 1 to 8 axes, got %d", axes);
  int64_t pairs = 0;
  for (int a = 0; a < axes; ++a) {
    if (dims[a] < 0 || dims[a] % 2 || dims[a] > 65536)
      return fail(CONVROT_ERR_INVALID, "an axis turns an even number of features, got %d", dims[a]);
    pairs += dims[a] / 2;
  }
  if (!(theta > 0.0)) return fail(CONVROT_ERR_INVALID, "theta must be positive");
  if (rows < 0) return fail(CONVROT_ERR_INVALID, "invalid shape rows=%lld", (long long)rows);
  if (rows == 0 || pairs == 0) return ok();
  if (rows > kMaxRows || rows * pairs > (int64_t(1) << 38)) return fail(CONVROT_ERR_UNSUPPORTED, "too many positions");
  if (!positions || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  return launch_status(convrot::launch_axes_table(positions, kind, rows, axes, dims, theta, out, (hipStream_t)stream),
                       "convrot_axes_table");
}

int convrot_qk_rotary(const void* q, const void* k, void* q_out, void* k_out, const int64_t* strides, int dtype,
                      int batch, int q_heads, int k_heads, int64_t length, int dim, const float* table, int pairs,
                      int64_t table_batch_stride, const void* q_weight, const void* k_weight, int weight_dtype,
                      float eps, int interleaved, void* stream) {
  if (int rc = check_rotary(dtype, batch, q_heads, k_heads, length, dim, table, pairs, table_batch_stride, q_weight,
                            k_weight, weight_dtype, strides))
    return rc;
  if (batch == 0 || length == 0 || dim == 0 || q_heads + k_heads == 0) return ok();
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)))
    return fail(CONVROT_ERR_INVALID, "null pointer argument");
  const convrot::RotaryShape sh{dtype,    batch,    q_heads,      k_heads, length,          dim, pairs, table, table_batch_stride,
                                q_weight, k_weight, weight_dtype, eps,     interleaved != 0};
  return launch_status(convrot::launch_qk_rotary(sh, q, k, q_out, k_out, strides, (hipStream_t)stream),
                       "convrot_qk_rotary");
}

int64_t convrot_qk_rotary_workspace_bytes(int dim) {
  return dim > 0 && dim <= 512 ? convrot::qk_rotary_workspace_bytes(dim) : 0;
}

int convrot_qk_rotary_backward(const void* dq, const void* dk, const void* q, const void* k, void* q_grad,
                               void* k_grad, void* q_weight_grad, void* k_weight_grad, const int64_t* strides,
                               int dtype, int batch, int q_heads, int k_heads, int64_t length, int dim,
                               const float* table, int pairs, int64_t table_batch_stride, const void* q_weight,
                               const void* k_weight, int weight_dtype, float eps, int interleaved, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  if (int rc = check_rotary(dtype, batch, q_heads, k_heads, length, dim, table, pairs, table_batch_stride, q_weight,
                            k_weight, weight_dtype, strides))
    return rc;
  if ((q_weight_grad && !q_weight) || (k_weight_grad && !k_weight))
    return fail(CONVROT_ERR_INVALID, "a weight's gradient needs the weight");
  if (batch == 0 || length == 0 || dim == 0 || q_heads + k_heads == 0) return ok();
  if ((q_heads && (!dq || !q_grad || (q_weight && !q))) || (k_heads && (!dk || !k_grad || (k_weight && !k))))
    return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if ((q_weight_grad || k_weight_grad) &&
      (!workspace || !aligned(workspace, 16) || workspace_bytes < convrot_qk_rotary_workspace_bytes(dim)))
    return fail(CONVROT_ERR_INVALID, "the rotary gradient needs a 16-byte aligned workspace of %lld bytes, got %lld",
                (long long)convrot_qk_rotary_workspace_bytes(dim), (long long)workspace_bytes);
  const convrot::RotaryShape sh{dtype,    batch,    q_heads,      k_heads, length,          dim, pairs, table, table_batch_stride,
                                q_weight, k_weight, weight_dtype, eps,     interleaved != 0};
  return launch_status(convrot::launch_qk_rotary_backward(sh, dq, dk, q, k, q_grad, k_grad, q_weight_grad,
                                                          k_weight_grad, strides, (float*)workspace,
                                                          (hipStream_t)stream),
                       "convrot_qk_rotary_backward");
}

// ---- linears in 8-bit floating point

namespace {

constexpr int64_t kMaxXsRow = int64_t(1) << 21;  // floats between rows' scales: a tile's offsets stay below 2^32

int64_t blocks_of(int64_t K) { return (K + convrot::kBlock - 1) / convrot::kBlock; }

int check_fp8_codes(const uint8_t* codes, int64_t stride, int64_t features, const float* scales) {
  if (!codes || !scales) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (stride < features || stride % 16 || !aligned(codes, 16) || !aligned(scales, 4))
    return fail(CONVROT_ERR_INVALID, "codes need 16-byte aligned rows of at least %lld bytes, got a stride of %lld",
                (long long)features, (long long)stride);
  if (stride > kMaxInt8Stride)
    return fail(CONVROT_ERR_UNSUPPORTED, "row strides of codes are limited to %lld bytes", (long long)kMaxInt8Stride);
  return ok();
}

// Checks of an FP8 product but for its activations; CONVROT_OK when the launch may proceed (M == 0 or
// N == 0 included).
int check_fp8(int64_t M, int64_t N, int64_t K, const uint8_t* weight, int64_t weight_stride, const float* wscales,
              int64_t wscales_stride, const void* out, int out_dtype) {
  if (!valid_dtype(out_dtype)) return fail(CONVROT_ERR_INVALID, "unsupported output dtype code %d", out_dtype);
  if (M < 0 || N < 0 || K <= 0)
    return fail(CONVROT_ERR_INVALID, "invalid GEMM shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if (K > kMaxFeatures)
    return fail(CONVROT_ERR_UNSUPPORTED, "FP8 GEMM supports K up to %lld, got %lld", (long long)kMaxFeatures, (long long)K);
  // 2^31 - 1 less what rounding a dimension up to whole tiles adds
  if (M > 0x7ffffe00 || N > 0x7ffffe00) return fail(CONVROT_ERR_UNSUPPORTED, "GEMM dimension too large");
  if (M == 0 || N == 0) return ok();
  if (!weight || !wscales || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (weight_stride < (K + 15) / 16 * 16 || weight_stride % 16 || !aligned(weight, 16) || !aligned(out, 16))
    return fail(CONVROT_ERR_INVALID,
                "FP8 operands need 16-byte aligned rows that cover K rounded up to 16 (K=%lld, weight stride %lld)",
                (long long)K, (long long)weight_stride);
  if (weight_stride > kMaxInt8Stride)
    return fail(CONVROT_ERR_UNSUPPORTED, "FP8 row strides are limited to %lld bytes", (long long)kMaxInt8Stride);
  if (wscales_stride < blocks_of(K) || !aligned(wscales, 4))
    return fail(CONVROT_ERR_INVALID, "weight scales need rows of %lld floats, got a stride of %lld",
                (long long)blocks_of(K), (long long)wscales_stride);
  return ok();
}

int check_fp8_work(const void* residual, const void* gate, int64_t rows_per_gate, const void* workspace,
                   int64_t workspace_bytes) {
  if (gate && !residual) return fail(CONVROT_ERR_INVALID, "a gate needs a residual");
  if (gate && rows_per_gate <= 0)
    return fail(CONVROT_ERR_INVALID, "rows_per_gate must be positive, got %lld", (long long)rows_per_gate);
  if (workspace_bytes < 0 || (workspace_bytes > 0 && !workspace))
    return fail(CONVROT_ERR_INVALID, "invalid workspace (%lld bytes)", (long long)workspace_bytes);
  if (workspace && !aligned(workspace, 256)) return fail(CONVROT_ERR_INVALID, "workspace must be 256-byte aligned");
  return ok();
}

// Codes and scales of rows in a scratch buffer: [rows][K rounded up to 128], then [blocks][rows rounded up to 4].
struct Fp8Scratch {
  uint8_t* codes;
  float* scales;
  int64_t stride, xs_block;
};
int64_t fp8_scratch_bytes(int64_t rows, int64_t K) {
  return rows <= 0 || K <= 0 ? 0 : rows * blocks_of(K) * convrot::kBlock + blocks_of(K) * ((rows + 3) / 4 * 4) * 4;
}
Fp8Scratch fp8_scratch(void* scratch, int64_t rows, int64_t K) {
  const int64_t stride = blocks_of(K) * convrot::kBlock;
  return {(uint8_t*)scratch, (float*)((uint8_t*)scratch + rows * stride), stride, (rows + 3) / 4 * 4};
}
int check_fp8_scratch(const void* scratch, int64_t bytes, int64_t rows, int64_t K) {
  if (!scratch || !aligned(scratch, 16) || bytes < fp8_scratch_bytes(rows, K))
    return fail(CONVROT_ERR_INVALID, "the FP8 linear needs a 16-byte aligned scratch buffer of %lld bytes, got %lld",
                (long long)fp8_scratch_bytes(rows, K), (long long)bytes);
  return ok();
}

}  // namespace

int convrot_quantize_fp8(const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride, uint8_t* codes,
                         int64_t codes_stride, float* scales, int64_t scales_row, int64_t scales_block, void* stream) {
  if (int rc = check_rows("8-bit quantization", x, dtype, rows, features, x_stride, kMaxFeatures)) return rc;
  if (rows == 0 || features == 0) return ok();
  if (int rc = check_fp8_codes(codes, codes_stride, features, scales)) return rc;
  if (scales_row < 1 || scales_block < 1)
    return fail(CONVROT_ERR_INVALID, "invalid strides of scales (%lld, %lld)", (long long)scales_row, (long long)scales_block);
  return launch_status(convrot::launch_quantize_fp8(x, dtype, rows, features, x_stride, codes, codes_stride, scales,
                                                    scales_row, scales_block, (hipStream_t)stream),
                       "convrot_quantize_fp8");
}

int convrot_quantize_fp8_weight(const void* w, int dtype, int64_t N, int64_t K, int64_t w_stride, uint8_t* codes,
                                int64_t codes_stride, float* scales, void* stream) {
  if (int rc = check_rows("8-bit quantization", w, dtype, N, K, w_stride, kMaxFeatures)) return rc;
  if (N == 0 || K == 0) return ok();
  if (int rc = check_fp8_codes(codes, codes_stride, K, scales)) return rc;
  return launch_status(convrot::launch_quantize_fp8_weight(w, dtype, N, K, w_stride, codes, codes_stride, scales,
                                                           (hipStream_t)stream),
                       "convrot_quantize_fp8_weight");
}

int convrot_fp8_gemm(const uint8_t* act, int64_t act_stride, const float* xscales, int64_t xscales_row,
                     int64_t xscales_block, const uint8_t* weight, int64_t weight_stride, const float* wscales,
                     int64_t wscales_stride, const float* bias, int64_t M, int64_t N, int64_t K, const void* residual,
                     const void* gate, int64_t gate_stride, int64_t rows_per_gate, void* workspace,
                     int64_t workspace_bytes, void* out, int out_dtype, void* stream) {
  if (int rc = check_fp8(M, N, K, weight, weight_stride, wscales, wscales_stride, out, out_dtype)) return rc;
  if (int rc = check_fp8_work(residual, gate, rows_per_gate, workspace, workspace_bytes)) return rc;
  if (M == 0 || N == 0) return ok();
  if (!act || !xscales) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (act_stride < (K + 15) / 16 * 16 || act_stride % 16 || !aligned(act, 16) || !aligned(xscales, 4))
    return fail(CONVROT_ERR_INVALID,
                "FP8 operands need 16-byte aligned rows that cover K rounded up to 16 (K=%lld, activation stride %lld)",
                (long long)K, (long long)act_stride);
  if (act_stride > kMaxInt8Stride)
    return fail(CONVROT_ERR_UNSUPPORTED, "FP8 row strides are limited to %lld bytes", (long long)kMaxInt8Stride);
  if (xscales_row < 0 || xscales_block < 0 || xscales_row > kMaxXsRow)
    return fail(CONVROT_ERR_UNSUPPORTED, "strides of activation scales (%lld, %lld) are not supported",
                (long long)xscales_row, (long long)xscales_block);
  convrot::GatedResidual gr{};
  if (residual)
    if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  const convrot::Fp8Operands p{act, weight, act_stride, weight_stride, xscales, wscales, bias, xscales_row,
                               xscales_block, wscales_stride, out, (int)M, (int)N, (int)K, gr, {}, 0, 0};
  const convrot::Workspace work{(uint8_t*)workspace, workspace ? (size_t)workspace_bytes : 0};
  return launch_status(convrot::launch_fp8_gemm(p, out_dtype, (hipStream_t)stream, work), "convrot_fp8_gemm");
}

int64_t convrot_fp8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > kMaxFeatures || M > 0x7ffffe00 || N > 0x7ffffe00) return 0;
  return convrot::fp8_workspace_bytes(M, N, K);
}

int64_t convrot_fp8_scratch_bytes(int64_t rows, int64_t K) { return fp8_scratch_bytes(rows, K); }

int convrot_fp8_linear(const void* x, int dtype, int64_t x_stride, const uint8_t* weight, int64_t weight_stride,
                       const float* wscales, int64_t wscales_stride, const float* bias, int64_t M, int64_t N,
                       int64_t K, const void* residual, const void* gate, int64_t gate_stride, int64_t rows_per_gate,
                       void* scratch, int64_t scratch_bytes, void* workspace, int64_t workspace_bytes, void* out,
                       void* stream) {
  if (int rc = check_rows("8-bit quantization", x, dtype, M, K, x_stride, kMaxFeatures)) return rc;
  if (int rc = check_fp8(M, N, K, weight, weight_stride, wscales, wscales_stride, out, dtype)) return rc;
  if (int rc = check_fp8_work(residual, gate, rows_per_gate, workspace, workspace_bytes)) return rc;
  if (M == 0 || N == 0) return ok();
  convrot::GatedResidual gr{};
  if (residual)
    if (int rc = check_residual(residual, gate, gate_stride, rows_per_gate, M, N, &gr)) return rc;
  const convrot::Workspace work{(uint8_t*)workspace, workspace ? (size_t)workspace_bytes : 0};
  // a fused launch's workgroups all read x: none may write into it
  const int64_t es = dtype == CONVROT_DTYPE_F32 ? 4 : 2;
  const uintptr_t xa = (uintptr_t)x, oa = (uintptr_t)out;
  const bool apart = oa + (uintptr_t)(M * N * es) <= xa || xa + (uintptr_t)(((M - 1) * x_stride + K) * es) <= oa;
  const bool fused = apart && convrot::fp8_fused(x, dtype, M, N, K, x_stride);
  if (!fused)
    if (int rc = check_fp8_scratch(scratch, scratch_bytes, M, K)) return rc;
  const Fp8Scratch c = fused ? Fp8Scratch{} : fp8_scratch(scratch, M, K);
  const convrot::Fp8Operands p{c.codes, weight, c.stride, weight_stride, c.scales, wscales, bias, 1,
                               c.xs_block, wscales_stride, out, (int)M, (int)N, (int)K, gr, {}, 0, 0};
  if (fused)
    return launch_status(convrot::launch_fp8_fused(p, x, x_stride, dtype, (hipStream_t)stream, work), "convrot_fp8_linear");
  hipError_t e = convrot::launch_quantize_fp8(x, dtype, M, K, x_stride, c.codes, c.stride, c.scales, 1, c.xs_block,
                                              (hipStream_t)stream);
  if (e == hipSuccess) e = convrot::launch_fp8_gemm(p, dtype, (hipStream_t)stream, work);
  return launch_status(e, "convrot_fp8_linear");
}

int convrot_fp8_fused(const void* x, int dtype, int64_t M, int64_t N, int64_t K, int64_t x_stride) {
  return M > 0 && N > 0 && K > 0 && valid_dtype(dtype) && convrot::fp8_fused(x, dtype, M, N, K, x_stride) ? 1 : 0;
}

namespace {

constexpr int64_t kMaxExperts = 65536;

// Checks of rows grouped by expert; `x_rows` is the number of rows of the activations.
int check_groups(const int32_t* offsets, int64_t experts, const int32_t* index, int64_t choices, int64_t x_rows,
                 int64_t rows) {
  if (experts < 1 || experts > kMaxExperts)
    return fail(CONVROT_ERR_UNSUPPORTED, "grouped products support 1 to %lld experts, got %lld", (long long)kMaxExperts,
                (long long)experts);
  if (x_rows < 0 || rows < 0 || choices < 1 || choices > 0x7fffffff)
    return fail(CONVROT_ERR_INVALID, "invalid groups of %lld rows of %lld (%lld choices)", (long long)rows,
                (long long)x_rows, (long long)choices);
  if (!index && x_rows != rows)
    return fail(CONVROT_ERR_INVALID, "%lld sorted rows, but %lld are grouped", (long long)x_rows, (long long)rows);
  if (rows > 0 && !offsets) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(offsets, 4) || !aligned(index, 4)) return fail(CONVROT_ERR_INVALID, "offsets and index must be aligned");
  return ok();
}

}  // namespace

int convrot_fp8_grouped_linear(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const uint8_t* weight,
                               int64_t weight_stride, int64_t weight_expert, const float* wscales,
                               int64_t wscales_stride, int64_t wscales_expert, const int32_t* offsets, int64_t experts,
                               const int32_t* index, int64_t choices, int64_t rows, int64_t N, int64_t K,
                               void* scratch, int64_t scratch_bytes, void* out, void* stream) {
  if (int rc = check_rows("8-bit quantization", x, dtype, x_rows, K, x_stride, kMaxFeatures)) return rc;
  if (int rc = check_fp8(rows, N, K, weight, weight_stride, wscales, wscales_stride, out, dtype)) return rc;
  if (int rc = check_groups(offsets, experts, index, choices, x_rows, rows)) return rc;
  if (weight_expert < 0 || weight_expert % 16 || wscales_expert < 0)
    return fail(CONVROT_ERR_INVALID, "experts' weights must be 16-byte aligned (%lld bytes apart)", (long long)weight_expert);
  if (rows == 0 || N == 0) return ok();
  if (x_rows > 0)
    if (int rc = check_fp8_scratch(scratch, scratch_bytes, x_rows, K)) return rc;
  const Fp8Scratch c = fp8_scratch(scratch, x_rows, K);
  if (index && (x_rows * c.stride > convrot::kMaxExtent || x_rows == 0))
    return fail(CONVROT_ERR_UNSUPPORTED, "rows read through an index support 1 to 2^32 codes, got %lld rows of %lld",
                (long long)x_rows, (long long)c.stride);
  const convrot::Fp8Operands p{c.codes, weight, c.stride, weight_stride, c.scales, wscales, nullptr, 1, c.xs_block,
                               wscales_stride, out, (int)rows, (int)N, (int)K, {},
                               {offsets, index, (int)experts, (int)choices, x_rows}, weight_expert, wscales_expert};
  hipError_t e = convrot::launch_quantize_fp8(x, dtype, x_rows, K, x_stride, c.codes, c.stride, c.scales, 1, c.xs_block,
                                              (hipStream_t)stream);
  if (e == hipSuccess) e = convrot::launch_fp8_gemm(p, dtype, (hipStream_t)stream, convrot::Workspace{});
  return launch_status(e, "convrot_fp8_grouped_linear");
}

// ---- what lies around the linears of a mixture of experts

namespace {

constexpr int64_t kMaxPlanExperts = 1024;  // one thread of the ordering workgroup each
constexpr int64_t kMaxRowFeatures = kMaxRows - 2047;  // a row is walked with 32 bits, up to 2048 features a step

int check_token_rows(const char* what, const void* y, int dtype, int64_t rows, int64_t features, int64_t stride,
                     int64_t tokens, int64_t choices) {
  if (int rc = check_rows(what, y, dtype, rows, features, stride, kMaxRowFeatures)) return rc;
  if (tokens < 0 || choices < 1 || tokens * choices > kMaxRows || choices > kMaxRows)
    return fail(CONVROT_ERR_INVALID, "%s: invalid shape of %lld tokens of %lld choices", what, (long long)tokens,
                (long long)choices);
  return ok();
}

}  // namespace

int64_t convrot_expert_plan_workspace_bytes(int64_t count, int64_t experts) {
  if (count <= 0 || count > kMaxRows || experts < 1 || experts > kMaxPlanExperts) return 0;
  return convrot::expert_plan_workspace_bytes(count, (int)experts);
}

int convrot_expert_plan(const void* ids, int ids_bits, int64_t count, int64_t experts, int32_t* offsets, int32_t* order,
                        int32_t* slots, void* workspace, int64_t workspace_bytes, void* stream) {
  if (ids_bits != 32 && ids_bits != 64) return fail(CONVROT_ERR_INVALID, "expert numbers have 32 or 64 bits, got %d", ids_bits);
  if (experts < 1 || experts > kMaxPlanExperts)
    return fail(CONVROT_ERR_UNSUPPORTED, "the order by expert supports 1 to %lld experts, got %lld",
                (long long)kMaxPlanExperts, (long long)experts);
  if (count < 0 || count > kMaxRows)
    return fail(CONVROT_ERR_UNSUPPORTED, "the order by expert supports at most 2^31-1 choices, got %lld", (long long)count);
  if (!offsets || (count > 0 && (!ids || !order || !slots))) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(ids, ids_bits / 8) || !aligned(offsets, 4) || !aligned(order, 4) || !aligned(slots, 4))
    return fail(CONVROT_ERR_INVALID, "expert numbers and their order must be aligned to their types");
  const int64_t need = convrot_expert_plan_workspace_bytes(count, experts);
  if (need > 0 && (!workspace || !aligned(workspace, 4) || workspace_bytes < need))
    return fail(CONVROT_ERR_INVALID, "the order by expert needs a workspace of %lld bytes, got %lld", (long long)need,
                (long long)workspace_bytes);
  return launch_status(convrot::launch_expert_plan(ids, ids_bits == 64, count, (int)experts, offsets, order, slots,
                                                   (int*)workspace, (hipStream_t)stream),
                       "convrot_expert_plan");
}

int convrot_gather_rows(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const int32_t* index,
                        int64_t choices, int64_t rows, int64_t features, void* out, void* stream) {
  if (int rc = check_rows("gathered rows", x, dtype, x_rows, features, x_stride, kMaxRowFeatures)) return rc;
  if (rows < 0 || rows > kMaxRows || choices < 1 || choices > kMaxRows)
    return fail(CONVROT_ERR_INVALID, "invalid shape of %lld gathered rows (%lld choices)", (long long)rows, (long long)choices);
  if (rows == 0 || features == 0) return ok();
  if (!index || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(index, 4) || !aligned(out, dtype == CONVROT_DTYPE_F32 ? 4 : 2))
    return fail(CONVROT_ERR_INVALID, "index and out must be aligned to their types");
  return launch_status(convrot::launch_gather_rows(x, dtype, x_rows, x_stride, index, (int)choices, rows, features, out,
                                                   (hipStream_t)stream),
                       "convrot_gather_rows");
}

int convrot_combine_rows(const void* y, int dtype, int64_t y_rows, int64_t y_stride, const int32_t* slots,
                         const float* weights, int64_t tokens, int64_t choices, int64_t features, void* out,
                         void* stream) {
  if (int rc = check_token_rows("combined rows", y, dtype, y_rows, features, y_stride, tokens, choices)) return rc;
  if (tokens == 0 || features == 0) return ok();
  if (!slots || !out) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(slots, 4) || !aligned(weights, 4) || !aligned(out, dtype == CONVROT_DTYPE_F32 ? 4 : 2))
    return fail(CONVROT_ERR_INVALID, "slots, weights and out must be aligned to their types");
  return launch_status(convrot::launch_combine_rows(y, dtype, y_rows, y_stride, slots, weights, tokens, (int)choices,
                                                    features, out, (hipStream_t)stream),
                       "convrot_combine_rows");
}

int convrot_combine_rows_backward(const void* dout, int64_t dout_stride, const void* y, int64_t y_stride, int dtype,
                                  int64_t y_rows, const int32_t* order, const int32_t* slots, const float* weights,
                                  int64_t tokens, int64_t choices, int64_t features, void* dy, float* dweights,
                                  void* stream) {
  if (int rc = check_token_rows("the gradient of combined rows", dout, dtype, tokens, features, dout_stride, tokens,
                                choices))
    return rc;
  if (y_rows != tokens * choices)
    return fail(CONVROT_ERR_INVALID, "%lld rows for %lld choices", (long long)y_rows, (long long)(tokens * choices));
  if (dweights)
    if (int rc = check_rows("the gradient of combined rows", y, dtype, y_rows, features, y_stride, kMaxRowFeatures)) return rc;
  if (tokens == 0 || (!dy && !dweights)) return ok();
  if (!slots || (dy && !order)) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(order, 4) || !aligned(slots, 4) || !aligned(weights, 4) || !aligned(dweights, 4) ||
      !aligned(dy, dtype == CONVROT_DTYPE_F32 ? 4 : 2))
    return fail(CONVROT_ERR_INVALID, "order, slots, weights and gradients must be aligned to their types");
  return launch_status(convrot::launch_combine_rows_backward(dout, dout_stride, y, y_stride, dtype, y_rows, order, slots,
                                                             weights, tokens, (int)choices, features, dy, dweights,
                                                             (hipStream_t)stream),
                       "convrot_combine_rows_backward");
}

// ---- grouped products in 16 bits

namespace {

// Checks of the operands of `rows` rows in 16 bits: [.., features], 16-byte aligned rows that cover them
// rounded up to 8.
int check_rows16(const char* what, const void* p, int64_t stride, int64_t features) {
  if (!p) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (!aligned(p, 16) || stride % 8 || stride < (features + 7) / 8 * 8)
    return fail(CONVROT_ERR_INVALID, "%s needs 16-byte aligned rows that cover %lld features rounded up to 8, got a stride of %lld",
                what, (long long)features, (long long)stride);
  if (stride * 2 > kMaxInt8Stride)
    return fail(CONVROT_ERR_UNSUPPORTED, "row strides are limited to %lld elements", (long long)(kMaxInt8Stride / 2));
  return ok();
}

int check_grouped(int dtype, const int32_t* offsets, int64_t experts, const int32_t* index, int64_t choices,
                  int64_t x_rows, int64_t rows, int64_t N, int64_t K) {
  if (dtype != CONVROT_DTYPE_F16 && dtype != CONVROT_DTYPE_BF16)
    return fail(CONVROT_ERR_INVALID, "grouped products take float16 or bfloat16, got dtype code %d", dtype);
  if (N < 1 || K < 1 || rows < 0)
    return fail(CONVROT_ERR_INVALID, "invalid grouped product rows=%lld N=%lld K=%lld", (long long)rows, (long long)N,
                (long long)K);
  if (N > kMaxFeatures || K > kMaxFeatures)
    return fail(CONVROT_ERR_UNSUPPORTED, "grouped products support up to %lld features, got N=%lld K=%lld",
                (long long)kMaxFeatures, (long long)N, (long long)K);
  if (rows > 0x7ffffe00) return fail(CONVROT_ERR_UNSUPPORTED, "GEMM dimension too large");
  return check_groups(offsets, experts, index, choices, x_rows, rows);
}

}  // namespace

int convrot_grouped_linear(const void* x, int dtype, int64_t x_rows, int64_t x_stride, const void* weight,
                           int64_t weight_stride, int64_t weight_expert, const int32_t* offsets, int64_t experts,
                           const int32_t* index, int64_t choices, int64_t rows, int64_t N, int64_t K, void* out,
                           void* stream) {
  if (int rc = check_grouped(dtype, offsets, experts, index, choices, x_rows, rows, N, K)) return rc;
  if (rows == 0) return ok();
  if (int rc = check_rows16("x", x, x_stride, K)) return rc;
  if (int rc = check_rows16("weight", weight, weight_stride, K)) return rc;
  if (weight_expert < 0 || weight_expert % 8 || !out || !aligned(out, 16))
    return fail(CONVROT_ERR_INVALID, "experts' weights and out must be 16-byte aligned");
  if (index && (x_rows == 0 || (x_rows - 1) * x_stride * 2 + (K + 7) / 8 * 16 > convrot::kMaxExtent))
    return fail(CONVROT_ERR_UNSUPPORTED, "rows read through an index support 1 to 2^32 bytes, got %lld rows %lld apart",
                (long long)x_rows, (long long)x_stride);
  const convrot::GroupedOperands p{(const uint16_t*)x, (const uint16_t*)weight, x_stride, weight_stride, weight_expert,
                                   (uint16_t*)out, (int)rows, (int)N, (int)K,
                                   {offsets, index, (int)experts, (int)choices, x_rows}};
  return launch_status(convrot::launch_grouped(index ? 1 : 0, p, dtype, (hipStream_t)stream), "convrot_grouped_linear");
}

int convrot_grouped_linear_rows_grad(const void* dy, int dtype, int64_t dy_stride, const void* weight,
                                     int64_t weight_stride, int64_t weight_expert, const int32_t* offsets,
                                     int64_t experts, int64_t rows, int64_t N, int64_t K, void* dx, void* stream) {
  if (int rc = check_grouped(dtype, offsets, experts, nullptr, 1, rows, rows, N, K)) return rc;
  if (rows == 0) return ok();
  if (int rc = check_rows16("dy", dy, dy_stride, N)) return rc;
  if (int rc = check_rows16("weight", weight, weight_stride, K)) return rc;
  if (weight_expert < 0 || weight_expert % 8 || !dx || !aligned(dx, 16))
    return fail(CONVROT_ERR_INVALID, "experts' weights and dx must be 16-byte aligned");
  const convrot::GroupedOperands p{(const uint16_t*)dy, (const uint16_t*)weight, dy_stride, weight_stride, weight_expert,
                                   (uint16_t*)dx, (int)rows, (int)K, (int)N, {offsets, nullptr, (int)experts, 1, rows}};
  return launch_status(convrot::launch_grouped(2, p, dtype, (hipStream_t)stream), "convrot_grouped_linear_rows_grad");
}

int convrot_grouped_linear_weight_grad(const void* dy, int dtype, int64_t dy_stride, const void* x, int64_t x_rows,
                                       int64_t x_stride, const int32_t* offsets, int64_t experts, const int32_t* index,
                                       int64_t choices, int64_t rows, int64_t N, int64_t K, void* dw, void* stream) {
  if (int rc = check_grouped(dtype, offsets, experts, index, choices, x_rows, rows, N, K)) return rc;
  if (!dw || !aligned(dw, 16)) return fail(CONVROT_ERR_INVALID, "dw must be 16-byte aligned");
  if (!offsets) return fail(CONVROT_ERR_INVALID, "null pointer argument");
  if (rows > 0) {
    if (int rc = check_rows16("dy", dy, dy_stride, N)) return rc;
    if (int rc = check_rows16("x", x, x_stride, K)) return rc;
    if (index && (x_rows == 0 || (x_rows - 1) * x_stride * 2 + (K + 7) / 8 * 16 > convrot::kMaxExtent))
      return fail(CONVROT_ERR_UNSUPPORTED, "rows read through an index support 1 to 2^32 bytes, got %lld rows %lld apart",
                  (long long)x_rows, (long long)x_stride);
  }
  const convrot::GroupedOperands p{(const uint16_t*)dy, (const uint16_t*)x, dy_stride, x_stride, 0, (uint16_t*)dw, (int)rows,
                                   (int)N, (int)K, {offsets, index, (int)experts, (int)choices, x_rows},
                                   convrot::Divisor((uint32_t)choices)};
  return launch_status(convrot::launch_grouped(index && rows > 0 ? 4 : 3, p, dtype, (hipStream_t)stream),
                       "convrot_grouped_linear_weight_grad");
}

}  // extern "C"
