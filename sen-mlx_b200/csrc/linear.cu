// linear.cu -- the C ABI of the 16-bit linear products (include/senmoe.h):
// argument checks, the choice of kernels, and the steps of the backward pass.

#include <cuda_runtime.h>

#include "../../include/senmoe.h"
#include "checks.h"
#include "kernels.h"
#include "linear.cuh"
#include "linear8.cuh"

using namespace senmoe;

namespace {

constexpr int64_t kMaxDim = int64_t(1) << 30;
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1024;  // row numbers, a tile past the last included, fit an int32

// A matrix operand: rows x cols, row stride in elements.
int check_matrix(const char* call, const char* name, const void* p, int64_t stride, int64_t cols) {
  if (!p) return reject(SENMOE_ERR_BAD_ARG, "%s: %s is NULL", call, name);
  if (reinterpret_cast<uintptr_t>(p) & 1) return reject(SENMOE_ERR_BAD_ARG, "%s: %s is not 2-byte aligned", call, name);
  if (stride < cols || stride > (int64_t(1) << 40))
    return reject(SENMOE_ERR_BAD_ARG, "%s: %s row stride %lld for rows of %lld elements", call, name,
                  (long long)stride, (long long)cols);
  return SENMOE_OK;
}

int check_vector(const char* call, const char* name, const void* p) {
  if (reinterpret_cast<uintptr_t>(p) & 1) return reject(SENMOE_ERR_BAD_ARG, "%s: %s is not 2-byte aligned", call, name);
  return SENMOE_OK;
}

// What forward and backward have in common; wide: rows of W.
int check_shape(const char* call, int32_t dtype, int32_t epilogue, int32_t groups, int32_t path, int64_t rows,
                int64_t in, int64_t out, const int32_t* offsets, int64_t* wide) {
  if (dtype != SENMOE_BF16 && dtype != SENMOE_FP16)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: dtype %d (bf16 and fp16 are supported)", call, dtype);
  if (epilogue < SENMOE_EPI_NONE || epilogue > SENMOE_EPI_GEGLU)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: epilogue %d", call, epilogue);
  if (path < SENMOE_LINEAR_AUTO || path > SENMOE_LINEAR_TCGEN05_SPLIT)
    return reject(SENMOE_ERR_BAD_ARG, "%s: path %d", call, path);
  if (groups < 1 || (!offsets && groups != 1))
    return reject(SENMOE_ERR_BAD_ARG, "%s: num_groups=%d%s", call, groups, offsets ? "" : " without offsets");
  if (groups > kMaxGroups) return reject(SENMOE_ERR_UNSUPPORTED, "%s: num_groups=%d (at most %d)", call, groups, kMaxGroups);
  if (reinterpret_cast<uintptr_t>(offsets) & 3) return reject(SENMOE_ERR_BAD_ARG, "%s: offsets is not 4-byte aligned", call);
  if (rows < 0 || rows > kMaxRows)
    return reject(SENMOE_ERR_BAD_ARG, "%s: rows=%lld", call, (long long)rows);
  *wide = epilogue >= SENMOE_EPI_SWIGLU ? 2 * out : out;
  if (in < 1 || out < 1 || in > kMaxDim || *wide > kMaxDim)
    return reject(SENMOE_ERR_BAD_ARG, "%s: in_features=%lld out_features=%lld", call, (long long)in, (long long)out);
  // the kernels count tiles, of 16 rows at least, in 32 bits, a grid past the last one included
  const int64_t cols = *wide > in ? *wide : in;
  if (((rows + 15) / 16 + groups) * ((cols + 63) / 64) >= (int64_t(1) << 30) ||
      groups * ((*wide + 63) / 64) * ((in + 63) / 64) >= (int64_t(1) << 30))
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: rows=%lld in_features=%lld out_features=%lld is too large", call,
                  (long long)rows, (long long)in, (long long)out);
  return SENMOE_OK;
}

int check_group_stride(const char* call, const char* name, int64_t group_stride, int64_t stride, int64_t rows,
                       int64_t cols, int groups) {
  if (groups > 1 && (group_stride < (rows - 1) * stride + cols || group_stride > (int64_t(1) << 44)))
    return reject(SENMOE_ERR_BAD_ARG, "%s: %s group stride %lld", call, name, (long long)group_stride);
  return SENMOE_OK;
}

// Whether the few-row kernel is the faster one.  Measured against the tcgen05
// tiles (us, W from HBM; bf16):
//   dense 2048 x 2048        8 rows 4.6 / 10.5   32 rows 7.0 / 10.7   64 rows 9.5 / 10.7
//   dense 2048 x 8192        8 rows 9.0 / 15.0   16 rows 11.1 / 14.9  32 rows 15.0 / 15.2
//   dense 2816 x 2112        32 rows 9.2 / 12.8  64 rows 12.2 / 12.6  96 rows 18.9 / 12.8
//   dense 512 x 2048         64 rows 4.6 / 7.5   96 rows 7.3 / 7.6
// Every 16-feature block reads all rows, so rows x W bounds it from 9 rows on.
//   128 experts, 2048 x 1536 swiglu:  8 rows 12.1 / 18.0  64 rows 59 / 63  128 rows 100 / 87
//   32 experts, the same:             128 rows 40.1 / 42.4  256 rows 52 / 42
//   128 experts, 768 x 2048:          8 rows 10.6 / 11.9  16 rows 17.4 / 16.1
// Grouped: with few rows a group, while the blocks are few or long (K).
bool few_rows(const LinearArgs& a) {
  if (!a.offsets)
    return a.rows <= 8 || (a.rows <= 64 && static_cast<int64_t>(a.n) * a.k * a.rows <= 400000000);
  if (a.rows > 64 && a.rows > 4 * a.groups) return false;
  const int64_t chunks = a.rows < a.groups ? a.rows : a.groups;
  return chunks * ((a.n + 15) / 16) <= (a.k >= 1024 ? 148 * 40 : 148 * 8);
}

int run_product(const char* call, const LinearArgs& a, LinearProduct p, int path, cudaStream_t st,
                const BiasJoin* bias = nullptr, bool* summed = nullptr) {
  // (no rows: dW's zeros, which no tile form is needed for)
  if (path == SENMOE_LINEAR_ANY || a.rows == 0) return cuda_status(call, launch_linear_any(a, p, st));
  const bool tc = linear_tc_supported(a, p);
  const bool force_tc = path >= SENMOE_LINEAR_TCGEN05 && path != SENMOE_LINEAR_SMALL;
  if (p == kProdForward && !force_tc) {
    const bool small = linear_small_supported(a);
    if (path == SENMOE_LINEAR_SMALL && !small)
      return reject(SENMOE_ERR_UNSUPPORTED, "%s: the few-row kernels need 16-byte aligned operands, in_features and "
                    "strides of a multiple of 8", call);
    if (small && (path == SENMOE_LINEAR_SMALL || few_rows(a))) return cuda_status(call, launch_linear_small(a, st));
  }
  if (force_tc && !tc)
    return reject(SENMOE_ERR_UNSUPPORTED, "%s: TMA needs 16-byte aligned operands, strides of a multiple of 8 elements",
                  call);
  const int form = path > SENMOE_LINEAR_SMALL ? path - SENMOE_LINEAR_SMALL : kFormAuto;
  return cuda_status(call, tc ? launch_linear_tc(a, p, form, bias, summed, st) : launch_linear_any(a, p, st));
}

int64_t round16(int64_t b) { return (b + 15) & ~int64_t(15); }

struct GradLayout {
  int64_t dz_stride = 0, dz_bytes = 0, partial_bytes = 0, max_bytes = 0;
  int run = 0;
  int64_t total() const { return dz_bytes + partial_bytes + max_bytes; }
};

GradLayout grad_layout(const SenMoeLinearGrad& g, int64_t wide) {
  GradLayout l;
  if (g.epilogue != SENMOE_EPI_NONE) {  // dz in rows that TMA can read
    l.dz_stride = (wide + 7) & ~int64_t(7);
    l.dz_bytes = round16(g.rows * l.dz_stride * 2);
    if (g.dtype == SENMOE_FP16 && g.rows > 0) l.max_bytes = round16(int64_t(g.num_groups) * 4);
  }
  l.run = dz_run(g.rows, g.offsets, g.epilogue);
  if (g.dbias) l.partial_bytes = round16(dz_slots(g.rows, g.num_groups, g.offsets, l.run) * wide * 4);
  return l;
}

}  // namespace

extern "C" {

int senmoe_linear(const SenMoeLinear* q, senmoe_stream_t stream) {
  clear_failure();
  const char* call = "linear";
  if (!q) return reject(SENMOE_ERR_BAD_ARG, "%s: product is NULL", call);
  int64_t wide = 0;
  int rc = check_shape(call, q->dtype, q->epilogue, q->num_groups, q->path, q->rows, q->in_features, q->out_features,
                       q->offsets, &wide);
  if (rc) return rc;
  if (q->rows == 0) return SENMOE_OK;
  if ((rc = check_matrix(call, "x", q->x, q->x_stride, q->in_features))) return rc;
  if ((rc = check_matrix(call, "weight", q->weight, q->weight_stride, q->in_features))) return rc;
  if ((rc = check_group_stride(call, "weight", q->weight_group_stride, q->weight_stride, wide, q->in_features,
                               q->num_groups)))
    return rc;
  if ((rc = check_matrix(call, "y", q->y, q->y_stride, q->out_features))) return rc;
  if (q->residual && (rc = check_matrix(call, "residual", q->residual, q->residual_stride, q->out_features))) return rc;
  if (q->preact && (rc = check_matrix(call, "preact", q->preact, q->preact_stride, wide))) return rc;
  if ((rc = check_vector(call, "bias", q->bias))) return rc;

  LinearArgs a{};
  a.a = q->x;
  a.a_stride = q->x_stride;
  a.b = q->weight;
  a.b_stride = q->weight_stride;
  a.b_group_stride = q->weight_group_stride;
  a.offsets = q->offsets;
  a.groups = q->num_groups;
  a.rows = q->rows;
  a.n = static_cast<int>(wide);
  a.k = static_cast<int>(q->in_features);
  a.act = q->epilogue;
  a.bias = q->bias;
  a.residual = q->residual;
  a.residual_stride = q->residual_stride;
  a.out = q->y;
  a.out_stride = q->y_stride;
  a.preact = q->preact;
  a.preact_stride = q->preact_stride;
  a.bf16 = q->dtype == SENMOE_BF16;
  return run_product(call, a, kProdForward, q->path, stream);
}

static int check_grad(const SenMoeLinearGrad* g, int64_t* wide) {
  const char* call = "linear_backward";
  if (!g) return reject(SENMOE_ERR_BAD_ARG, "%s: grad is NULL", call);
  return check_shape(call, g->dtype, g->epilogue, g->num_groups, g->path, g->rows, g->in_features, g->out_features,
                     g->offsets, wide);
}

int64_t senmoe_linear_backward_workspace(const SenMoeLinearGrad* g) {
  clear_failure();
  int64_t wide = 0;
  const int rc = check_grad(g, &wide);
  return rc ? -int64_t(rc) : grad_layout(*g, wide).total();
}

int senmoe_linear_backward(const SenMoeLinearGrad* g, senmoe_stream_t stream) {
  clear_failure();
  const char* call = "linear_backward";
  int64_t wide = 0;
  int rc = check_grad(g, &wide);
  if (rc) return rc;
  const bool some = g->rows > 0, act = g->epilogue != SENMOE_EPI_NONE;
  const int E = g->num_groups;
  if (some && (rc = check_matrix(call, "dy", g->dy, g->dy_stride, g->out_features))) return rc;
  if (some && act && (rc = check_matrix(call, "preact", g->preact, g->preact_stride, wide))) return rc;
  if (some && g->dx) {
    if ((rc = check_matrix(call, "dx", g->dx, g->dx_stride, g->in_features))) return rc;
    if ((rc = check_matrix(call, "weight", g->weight, g->weight_stride, g->in_features))) return rc;
    if ((rc = check_group_stride(call, "weight", g->weight_group_stride, g->weight_stride, wide, g->in_features, E)))
      return rc;
  }
  if (g->dweight) {
    if (some && (rc = check_matrix(call, "x", g->x, g->x_stride, g->in_features))) return rc;
    if ((rc = check_matrix(call, "dweight", g->dweight, g->dweight_stride, g->in_features))) return rc;
    if ((rc = check_group_stride(call, "dweight", g->dweight_group_stride, g->dweight_stride, wide, g->in_features, E)))
      return rc;
  }
  if ((rc = check_vector(call, "dbias", g->dbias))) return rc;
  const GradLayout l = grad_layout(*g, wide);
  if (l.total() > 0 && (!g->workspace || g->workspace_bytes < l.total()))
    return reject(SENMOE_ERR_BAD_ARG, "%s: workspace of %lld bytes, %lld needed", call,
                  g->workspace ? (long long)g->workspace_bytes : 0ll, (long long)l.total());
  if (reinterpret_cast<uintptr_t>(g->workspace) & 15)
    return reject(SENMOE_ERR_BAD_ARG, "%s: workspace is not 16-byte aligned", call);

  LinearGradArgs ga{};
  ga.dy = g->dy;
  ga.dy_stride = g->dy_stride;
  ga.preact = g->preact;
  ga.preact_stride = g->preact_stride;
  ga.offsets = g->offsets;
  ga.groups = E;
  ga.rows = g->rows;
  ga.n = static_cast<int>(wide);
  ga.act = g->epilogue;
  ga.dz = g->workspace;
  ga.dz_stride = l.dz_stride;
  ga.dbias = g->dbias;
  ga.run = l.run;
  if (l.partial_bytes) ga.partial = reinterpret_cast<float*>(static_cast<char*>(g->workspace) + l.dz_bytes);
  if (l.max_bytes && (g->dx || g->dweight))
    ga.dz_max = reinterpret_cast<unsigned*>(static_cast<char*>(g->workspace) + l.dz_bytes + l.partial_bytes);
  ga.bf16 = g->dtype == SENMOE_BF16;
  if (act && (rc = cuda_status(call, launch_dz(ga, stream)))) return rc;
  BiasJoin join{act ? ga.partial : nullptr, g->offsets, E, l.run, ga.n, g->rows, g->dbias};
  bool summed = !g->dbias || (act && some && !ga.partial);  // no bias gradient, or there already

  LinearArgs a{};
  a.a = act ? ga.dz : g->dy;
  a.a_stride = act ? l.dz_stride : g->dy_stride;
  a.offsets = g->offsets;
  a.groups = E;
  a.rows = g->rows;
  a.n = static_cast<int>(wide);
  a.k = static_cast<int>(g->in_features);
  a.bf16 = ga.bf16;
  a.dz_max = ga.dz_max;
  if (some && g->dx) {
    a.b = g->weight;
    a.b_stride = g->weight_stride;
    a.b_group_stride = g->weight_group_stride;
    a.out = g->dx;
    a.out_stride = g->dx_stride;
    if ((rc = run_product(call, a, kProdInput, g->path, stream))) return rc;
  }
  if (g->dweight) {
    a.b = g->x;
    a.b_stride = g->x_stride;
    a.out = g->dweight;
    a.out_stride = g->dweight_stride;
    a.out_group_stride = g->dweight_group_stride;
    if ((rc = run_product(call, a, kProdWeight, g->path, stream, summed ? nullptr : &join, &summed))) return rc;
  }
  if (!summed) {  // no dweight, or a form that does not take it
    if (!act && (rc = cuda_status(call, launch_dz(ga, stream)))) return rc;
    join.partial = ga.partial;
    if ((act || ga.partial || !some) && (rc = cuda_status(call, launch_bias_join(join, ga.bf16, stream)))) return rc;
  }
  return SENMOE_OK;
}

int senmoe_linear_check(senmoe_stream_t stream) {
  clear_failure();
  int error = 0, *word8 = nullptr;
  int rc = cuda_status("linear_check", linear8_error_word(&word8));
  if (rc || (rc = cuda_status("linear_check", linear_device_error(stream, &error, word8)))) return rc;
  if (error == kDevWaitTimeout) return reject(SENMOE_ERR_TIMEOUT, "linear: a bounded wait on the device ran out");
  return error ? reject(SENMOE_ERR_DEVICE, "linear: device error %d", error) : SENMOE_OK;
}

int senmoe_selftest_linear_wait(senmoe_stream_t stream) {
  clear_failure();
  return cuda_status("selftest_linear_wait", selftest_linear_wait(stream));
}

}  // extern "C"
