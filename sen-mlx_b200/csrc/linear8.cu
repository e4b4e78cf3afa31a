// linear8.cu -- the C ABI of rows in 8 bits and the products over them
// (include/senmoe.h): argument checks and the choice of kernels.

#include <cuda_runtime.h>

#include "checks.h"
#include "linear8.cuh"

using namespace senmoe;

namespace {

constexpr int64_t kMaxDim = int64_t(1) << 30;
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1024;  // row numbers, a tile past the last included, fit an int32
constexpr int64_t kMaxStride = int64_t(1) << 40;

// A matrix of 16-bit elements, row stride in elements.
int check_matrix(const char* call, const char* name, const void* p, int64_t stride, int64_t cols) {
  if (!p) return reject(SENMOE_ERR_BAD_ARG, "%s: %s is NULL", call, name);
  if (reinterpret_cast<uintptr_t>(p) & 1) return reject(SENMOE_ERR_BAD_ARG, "%s: %s is not 2-byte aligned", call, name);
  if (stride < cols || stride > kMaxStride)
    return reject(SENMOE_ERR_BAD_ARG, "%s: %s row stride %lld for rows of %lld elements", call, name,
                  (long long)stride, (long long)cols);
  return SENMOE_OK;
}

// Rows in 8 bits: codes on a 16-byte grid, scales anywhere.
int check_rows8(const char* call, const char* name, const void* codes, int64_t stride, const void* scales,
                int64_t scales_stride, int64_t cols) {
  if (!codes || !scales) return reject(SENMOE_ERR_BAD_ARG, "%s: %s or its scales are NULL", call, name);
  if (stride < cols || stride > (int64_t(1) << 36) || scales_stride < cols / kBlock8 || scales_stride > kMaxStride)
    return reject(SENMOE_ERR_BAD_ARG, "%s: %s row strides %lld and %lld for rows of %lld elements", call, name,
                  (long long)stride, (long long)scales_stride, (long long)cols);
  if ((reinterpret_cast<uintptr_t>(codes) | stride) & 15)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: %s codes are not on a 16-byte grid", call, name);
  return SENMOE_OK;
}

int check_type(const char* call, int32_t dtype, int32_t epilogue) {
  if (dtype != SENMOE_BF16 && dtype != SENMOE_FP16)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: dtype %d (bf16 and fp16 are supported)", call, dtype);
  if (epilogue < SENMOE_EPI_NONE || epilogue > SENMOE_EPI_GEGLU)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: epilogue %d", call, epilogue);
  return SENMOE_OK;
}

// Whether the few-row kernel is the faster one.  Measured against the tcgen05
// tiles (us, W from HBM):
//   dense 2048 x 2048    8 rows 4.7 / 8.9    16 rows 5.8 / 9.3    64 rows 13.9 / 9.5
//   dense 2816 x 2112    8 rows 5.8 / 10.7   16 rows 7.4 / 10.7   32 rows 10.7 / 10.8
//   dense 512 x 2048     8 rows 2.4 / 6.1    64 rows 5.9 / 6.3    96 rows 10.2 / 6.4
//   dense 2048 x 8192    8 rows 10.9 / 10.0  8192 x 2048  1 row 12.6 / 12.6
//   dense 1024 x 512     64 rows 8.1 / 7.2   4096 x 512   8 rows 7.0 / 9.7   16 rows 9.3 / 9.7
// A block walks the whole of K for all rows, whatever the number of blocks.
// It reads W in pieces of 32 bytes a row, which bounds it at 2 TB/s, and all
// rows for every 16 features; and its blocks, short ones, should be resident
// together.  Grouped (touched experts x K x rows of W), by what the experts hold,
// and blocks:
//   8 x 768 x 2048    1024 blocks 12.9 / 9.4    8 x 2048 x 1536 (8 bits) 192 blocks 14.0 / 13.0
//   4 x 2048 x 1536 (8 bits)  96 blocks 10.4 / 11.8    8 x 512 x 1024  512 blocks 6.4 / 8.3
//   16 x 96 x 512     512 blocks 6.3 / 7.7      32 x 256 x 512   1024 blocks 10.6 / 8.4
// and with more than 8 rows a group, where an SM has one block (two of 16 rows
// with a 16-bit output) and K times a chunk's rows counts, twice with an 8-bit
// output's larger blocks, four times with a gated pair's, half as many warps of
// which share K:
//   2 x 2048 x 1536  16 rows 8.4 / 11.2  21 rows (192 blocks) 15.6 / 11.3
//   2 x 4096 x 512   16 rows 10.4 / 11.6  32 rows 14.4 / 11.7
//   2 x 2816 x 704 geglu  32 rows 10.6 / 12.5   4 x 768 x 2048  16 rows (512 blocks) 10.0 / 9.2
//   8 bits: 2 x 1024 x 1536  32 rows 8.3 / 9.5  2 x 2048 x 1024  16 rows 8.8 / 11.2  32 rows 12.8 / 11.4
//   8 bits, swiglu: 3 x 1024 x 1024  16 rows 8.4 / 9.7  21 rows 11.3 / 9.8  2 x 2048 x 1536  12 rows 13.6 / 11.9
bool few_rows8(const Linear8Args& a) {
  const int64_t weight = static_cast<int64_t>(a.n) * a.k;
  const int64_t chunks = !a.offsets ? (a.rows + 63) / 64 : a.rows < a.groups ? a.rows : a.groups;
  const int rows_of_w = !a.codes ? 16 : act_gated(a.act) ? 64 : 32;  // of a block
  const int64_t blocks = chunks * ((a.n + rows_of_w - 1) / rows_of_w);
  if (a.rows > 64 || blocks > 148 * 4) return false;
  if (a.offsets) {
    const int chunk = linear8_small_chunk(a);
    if (chunk > 8 && (blocks > (chunk == 16 && !a.codes ? 2 : 1) * 148 ||
                      static_cast<int64_t>(a.k) * chunk > 95000 / (!a.codes ? 1 : act_gated(a.act) ? 4 : 2)))
      return false;
    return weight * chunks <= 13000000;
  }
  const int64_t each = a.rows > 8 ? a.rows : 8;
  return weight * each <= 100000000 && a.k * each <= 50000;
}

}  // namespace

extern "C" {

int senmoe_quantize8(const SenMoeQuantize8* q, senmoe_stream_t stream) {
  clear_failure();
  const char* call = "quantize8";
  if (!q) return reject(SENMOE_ERR_BAD_ARG, "%s: quantize is NULL", call);
  int rc = check_type(call, q->dtype, q->epilogue);
  if (rc) return rc;
  const int64_t wide = q->epilogue >= SENMOE_EPI_SWIGLU ? 2 * q->n : q->n;
  if (q->rows < 0 || q->rows > kMaxRows || q->n < 1 || wide > kMaxDim)
    return reject(SENMOE_ERR_BAD_ARG, "%s: rows=%lld n=%lld", call, (long long)q->rows, (long long)q->n);
  if (q->n % kBlock8) return reject(SENMOE_ERR_UNSUPPORTED, "%s: n=%lld (a multiple of %d)", call, (long long)q->n, kBlock8);
  if (q->rows == 0) return SENMOE_OK;
  if ((rc = check_matrix(call, "x", q->x, q->x_stride, q->n))) return rc;
  if (q->epilogue && (rc = check_matrix(call, "preact", q->preact, q->preact_stride, wide))) return rc;
  if ((rc = check_rows8(call, "codes", q->codes, q->codes_stride, q->scales, q->scales_stride, wide))) return rc;
  Quantize8Args a{};
  a.x = q->x;
  a.x_stride = q->x_stride;
  a.preact = q->preact;
  a.preact_stride = q->preact_stride;
  a.rows = q->rows;
  a.n = static_cast<int>(q->n);
  a.act = q->epilogue;
  a.bf16 = q->dtype == SENMOE_BF16;
  a.codes = static_cast<uint8_t*>(q->codes);
  a.codes_stride = q->codes_stride;
  a.scales = static_cast<uint8_t*>(q->scales);
  a.scales_stride = q->scales_stride;
  return cuda_status(call, launch_quantize8(a, stream));
}

int senmoe_linear8(const SenMoeLinear8* q, senmoe_stream_t stream) {
  clear_failure();
  const char* call = "linear8";
  if (!q) return reject(SENMOE_ERR_BAD_ARG, "%s: product is NULL", call);
  int rc = check_type(call, q->dtype, q->epilogue);
  if (rc) return rc;
  const int groups = q->num_groups;
  if (q->path < SENMOE_LINEAR_AUTO || q->path > SENMOE_LINEAR_TCGEN05_SPLIT)
    return reject(SENMOE_ERR_BAD_ARG, "%s: path %d", call, q->path);
  if (q->path == SENMOE_LINEAR_ANY) return reject(SENMOE_ERR_UNSUPPORTED, "%s: path %d", call, q->path);
  if (groups < 1 || (!q->offsets && groups != 1))
    return reject(SENMOE_ERR_BAD_ARG, "%s: num_groups=%d%s", call, groups, q->offsets ? "" : " without offsets");
  if (groups > kMaxGroups) return reject(SENMOE_ERR_UNSUPPORTED, "%s: num_groups=%d (at most %d)", call, groups, kMaxGroups);
  if (reinterpret_cast<uintptr_t>(q->offsets) & 3)
    return reject(SENMOE_ERR_BAD_ARG, "%s: offsets is not 4-byte aligned", call);
  if (q->rows < 0 || q->rows > kMaxRows) return reject(SENMOE_ERR_BAD_ARG, "%s: rows=%lld", call, (long long)q->rows);
  const int64_t in = q->in_features, out = q->out_features;
  const int64_t wide = q->epilogue >= SENMOE_EPI_SWIGLU ? 2 * out : out;
  if (in < 1 || out < 1 || in > kMaxDim || wide > kMaxDim)
    return reject(SENMOE_ERR_BAD_ARG, "%s: in_features=%lld out_features=%lld", call, (long long)in, (long long)out);
  if (in % kBlock8)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: in_features=%lld (a multiple of %d)", call, (long long)in, kBlock8);
  // the kernels count tiles, of 16 rows at least, in 32 bits, a grid past the last one included
  if (((q->rows + 15) / 16 + groups) * ((wide + 15) / 16) >= (int64_t(1) << 30))
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: rows=%lld out_features=%lld is too large", call, (long long)q->rows,
                  (long long)out);
  if (!q->y == !q->y_codes && q->rows > 0)
    return reject(SENMOE_ERR_BAD_ARG, "%s: y and y_codes: one of the two", call);
  if (q->y_codes && out % kBlock8)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: out_features=%lld in 8 bits (a multiple of %d)", call, (long long)out, kBlock8);
  if (q->rows == 0) return SENMOE_OK;
  if ((rc = check_rows8(call, "x", q->x, q->x_stride, q->x_scales, q->x_scales_stride, in))) return rc;
  if ((rc = check_rows8(call, "weight", q->weight, q->weight_stride, q->weight_scales, q->weight_scales_stride, in)))
    return rc;
  if (groups > 1) {
    const int64_t gs = q->weight_group_stride, ss = q->weight_scales_group_stride;
    if (gs < (wide - 1) * q->weight_stride + in || gs >= (int64_t(1) << 39) ||
        ss < (wide - 1) * q->weight_scales_stride + in / kBlock8 || ss > kMaxStride)
      return reject(SENMOE_ERR_BAD_ARG, "%s: weight group strides %lld and %lld", call, (long long)gs, (long long)ss);
    if (gs & 15) return reject(SENMOE_ERR_UNSUPPORTED, "%s: weight codes are not on a 16-byte grid", call);
  }
  if (q->y && (rc = check_matrix(call, "y", q->y, q->y_stride, out))) return rc;
  if (q->y_codes && (rc = check_rows8(call, "y", q->y_codes, q->y_codes_stride, q->y_scales, q->y_scales_stride, out)))
    return rc;
  if (q->residual && (rc = check_matrix(call, "residual", q->residual, q->residual_stride, out))) return rc;
  if (q->preact && (rc = check_matrix(call, "preact", q->preact, q->preact_stride, wide))) return rc;
  if (reinterpret_cast<uintptr_t>(q->bias) & 1) return reject(SENMOE_ERR_BAD_ARG, "%s: bias is not 2-byte aligned", call);

  Linear8Args a{};
  a.x = static_cast<const uint8_t*>(q->x);
  a.x_stride = q->x_stride;
  a.x_scales = static_cast<const uint8_t*>(q->x_scales);
  a.x_scales_stride = q->x_scales_stride;
  a.w = static_cast<const uint8_t*>(q->weight);
  a.w_stride = q->weight_stride;
  a.w_group_stride = groups > 1 ? q->weight_group_stride : 0;
  a.w_scales = static_cast<const uint8_t*>(q->weight_scales);
  a.w_scales_stride = q->weight_scales_stride;
  a.w_scales_group_stride = groups > 1 ? q->weight_scales_group_stride : 0;
  a.offsets = q->offsets;
  a.groups = groups;
  a.rows = q->rows;
  a.n = static_cast<int>(wide);
  a.k = static_cast<int>(in);
  a.act = q->epilogue;
  a.bf16 = q->dtype == SENMOE_BF16;
  a.bias = q->bias;
  a.residual = q->residual;
  a.residual_stride = q->residual_stride;
  a.y = q->y;
  a.y_stride = q->y_stride;
  a.codes = static_cast<uint8_t*>(q->y_codes);
  a.codes_stride = q->y_codes_stride;
  a.scales = static_cast<uint8_t*>(q->y_scales);
  a.scales_stride = q->y_scales_stride;
  a.preact = q->preact;
  a.preact_stride = q->preact_stride;
  const bool small = linear8_small_supported(a);
  if (q->path == SENMOE_LINEAR_SMALL && !small)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: %lld rows on the few-row kernels", call, (long long)q->rows);
  if (q->path == SENMOE_LINEAR_SMALL || (q->path == SENMOE_LINEAR_AUTO && small && few_rows8(a)))
    return cuda_status(call, launch_linear8_small(a, stream));
  const int form = q->path > SENMOE_LINEAR_SMALL ? q->path - SENMOE_LINEAR_SMALL : kFormAuto;
  return cuda_status(call, launch_linear8_tc(a, form, stream));
}

}  // extern "C"
