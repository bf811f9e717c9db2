// Residual norm: checks, shapes and the C entry points (kernels: residual_norm_forward.cuh, residual_norm_backward.cuh).
#include "residual_norm.cuh"

namespace opus {

int check_norm(const char* what, const opus_residual_norm_args* a) {
  if (a == nullptr) return set_error(OPUS_ERR_INVALID, "%s: NULL arguments", what);
  if (a->rows < 0 || a->d < 1) return set_error(OPUS_ERR_INVALID, "%s: bad sizes rows=%lld d=%d", what, (long long)a->rows, a->d);
  if (a->d > kNormMaxWidth) return set_error(OPUS_ERR_UNSUPPORTED, "%s: d up to %d (got %d)", what, kNormMaxWidth, a->d);
  if (a->kind != 0 && a->kind != 1) return set_error(OPUS_ERR_INVALID, "%s: kind %d is neither 0 (RMS) nor 1 (layer)", what, a->kind);
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->y_dtype) || (a->x_dtype != a->y_dtype && a->x_dtype != OPUS_DTYPE_F32))
    return set_error(OPUS_ERR_UNSUPPORTED, "%s: x is of y's type (bf16, f16 or f32) or f32", what);
  if (a->post && a->y == nullptr && a->rows > 0) return set_error(OPUS_ERR_INVALID, "%s: a norm after the block needs y", what);
  if (!a->post && (a->post_weight || a->post_bias))
    return set_error(OPUS_ERR_INVALID, "%s: post_weight and post_bias belong to post", what);
  const void* p[5] = {a->weight, a->bias, a->post_weight, a->post_bias, a->gate};
  const int t[5] = {a->weight_dtype, a->bias_dtype, a->post_weight_dtype, a->post_bias_dtype, a->gate_dtype};
  for (int i = 0; i < 5; ++i) {
    if (p[i] == nullptr) continue;
    if (!dtype_ok(t[i])) return set_error(OPUS_ERR_UNSUPPORTED, "%s: a parameter is neither bf16, f16 nor f32", what);
    if (reinterpret_cast<uintptr_t>(p[i]) % dtype_bytes(t[i]) != 0)
      return set_error(OPUS_ERR_INVALID, "%s: a parameter is not aligned to its elements", what);
  }
  if (a->gate != nullptr) {
    if (a->y == nullptr && a->rows > 0) return set_error(OPUS_ERR_INVALID, "%s: a gate needs y", what);
    if (a->gate_rows < 1 || a->rows % a->gate_rows != 0)
      return set_error(OPUS_ERR_INVALID, "%s: %lld rows cannot share %lld gate rows evenly", what, (long long)a->rows,
                       (long long)a->gate_rows);
  }
  return OPUS_OK;
}

// Vector loads of the parameters need their arrays on 16-byte boundaries.
bool norm_params_aligned(const opus_residual_norm_args* a) {
  const void* p[5] = {a->weight, a->bias, a->post_weight, a->post_bias, a->gate};
  for (const void* q : p)
    if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return false;
  return true;
}

// The launch's shape for vectors of V elements, at most `most` of them (a power of two) a thread: as few threads
// a row as that allows, and as many rows as a block of `threads` holds.  Returns how many vectors a thread (a power of two) those threads need.
int norm_shape(const opus_residual_norm_args* a, int V, int most, NormShape* s, int threads) {
  const int full = (a->d + V - 1) / V;
  int group = 1;
  while (group < 32 && group * most < full) group <<= 1;
  if (group * most < full) group = ((full + most - 1) / most + 31) / 32 * 32;
  // rows of less than a warp: a vector for each lane, so that its loads are neighbours
  while (group < 32 && group < full) group <<= 1;
  int k = 1;
  while (k * group < full) k <<= 1;
  s->rows = a->rows;
  s->seq = a->gate != nullptr && a->gate_rows > 1 ? a->rows / a->gate_rows : a->rows;
  if (s->seq < 1) s->seq = 1;
  s->d = a->d;
  s->group = group;
  s->groups = group >= threads ? 1 : threads / group;
  s->ranks = 1;
  s->err = nullptr;
  s->layer = a->kind;
  s->eps = a->eps;
  s->blocks = 0;
  return k;
}

// Of rows wider than a block of NV vectors a thread: a cluster of as few blocks (2, 4 or 8) as hold a row, and as few
// threads in each as share it evenly (more than 64, since half as many full blocks would not have held it).
int norm_shape_wide(const opus_residual_norm_args* a, int V, int NV, NormShape* s) {
  norm_shape(a, V, NV, s);
  const int full = (a->d + V - 1) / V;
  int ranks = 2;
  while (ranks * kNormThreads * NV < full) ranks *= 2;
  s->group = ((full + ranks * NV - 1) / (ranks * NV) + 31) / 32 * 32;
  s->groups = 1;
  s->ranks = ranks;
  s->err = device_error_word();
  return s->err != nullptr ? OPUS_OK : set_error(OPUS_ERR_CUDA, "device error word unavailable");
}

namespace {

bool on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace
}  // namespace opus

using namespace opus;

extern "C" int opus_residual_norm(const opus_residual_norm_args* args, void* stream) {
  int rc = check_norm("residual_norm", args);
  if (rc) return rc;
  opus_residual_norm_args a = *args;
  if (a.rows == 0) return OPUS_OK;
  if (!a.x || !a.n || !a.stats) return set_error(OPUS_ERR_INVALID, "residual_norm: NULL pointer");
  if (!a.h && (a.y || a.residual_scale != 1.0f))
    return set_error(OPUS_ERR_INVALID, "residual_norm: h is NULL, and differs from x");
  const int xb = dtype_bytes(a.x_dtype), yb = dtype_bytes(a.y_dtype);
  if (a.x_stride < a.d || (a.y && a.y_stride < a.d)) return set_error(OPUS_ERR_INVALID, "residual_norm: row stride < d");
  if (!on(a.x, xb) || !on(a.h, xb) || !on(a.y, yb) || !on(a.n, yb) || !on(a.stats, 16))
    return set_error(OPUS_ERR_INVALID, "residual_norm: a pointer is not aligned to its elements");
  const int V = 16 / xb;
  const bool vec = norm_params_aligned(&a) && a.d % V == 0 && a.x_stride % V == 0 && on(a.x, 16) && on(a.h, 16) && on(a.n, V * yb) &&
                   (!a.y || (a.y_stride % V == 0 && on(a.y, V * yb)));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a.x_dtype == OPUS_DTYPE_F32) {
    if (a.y_dtype == OPUS_DTYPE_F32) return residual_norm_f32(a, vec, st);
    if (a.y_dtype == OPUS_DTYPE_F16) return residual_norm_f32_f16(a, vec, st);
    return residual_norm_f32_bf16(a, vec, st);
  }
  if (a.x_dtype == OPUS_DTYPE_F16) return residual_norm_f16(a, vec, st);
  return residual_norm_bf16(a, vec, st);
}

extern "C" int64_t opus_residual_norm_grad_workspace_bytes(const opus_residual_norm_args* a) {
  if (a == nullptr || a->rows <= 0 || a->d < 1) return 256;
  const int64_t samples = a->gate != nullptr && a->gate_rows > 1 && a->rows % a->gate_rows == 0 ? a->gate_rows : 0;
  // a block holds at most 256 rows, and no more blocks run than there are rows
  int64_t blocks = static_cast<int64_t>(sm_count()) * kGradBlocksPerSm;
  blocks = blocks < a->rows ? blocks : a->rows;
  int64_t workers = 0;
  if (samples > 0) {
    workers = blocks * (a->d > 2048 ? 1 : a->d > 256 ? 8 : 256);
    workers = (workers < a->rows + 256 ? workers : a->rows + 256) + samples;
  }
  return align256((blocks * kColumns + workers) * a->d * 4);
}

extern "C" int opus_residual_norm_grad(const opus_residual_norm_args* args, void* workspace, int64_t workspace_bytes,
                                       void* stream) {
  int rc = check_norm("residual_norm_grad", args);
  if (rc) return rc;
  const opus_residual_norm_args& a = *args;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  void* outs[kColumns] = {a.grad_weight, a.grad_bias, a.grad_post_weight, a.grad_post_bias, a.grad_gate};
  const void* of[kColumns] = {a.weight, a.bias, a.post_weight, a.post_bias, a.gate};
  const int types[kColumns] = {a.weight_dtype, a.bias_dtype, a.post_weight_dtype, a.post_bias_dtype, a.gate_dtype};
  int wanted = 0;
  for (int c = 0; c < kColumns; ++c) {
    if (outs[c] == nullptr) continue;
    if (of[c] == nullptr) return set_error(OPUS_ERR_INVALID, "residual_norm_grad: a gradient of no parameter");
    if (!on(outs[c], dtype_bytes(types[c])))
      return set_error(OPUS_ERR_INVALID, "residual_norm_grad: a pointer is not aligned to its elements");
    wanted |= 1 << c;
    if (a.rows == 0)
      OPUS_CUDA_TRY(cudaMemsetAsync(outs[c], 0, (c == kGate ? a.gate_rows : 1) * static_cast<int64_t>(a.d) * dtype_bytes(types[c]), st));
  }
  if (a.rows == 0) return OPUS_OK;
  if (!a.h || !a.stats || !a.grad_x || (!a.grad_n && !a.grad_h) || (a.y != nullptr && a.grad_y == nullptr) ||
      (a.y == nullptr && a.grad_y != nullptr) || !workspace)
    return set_error(OPUS_ERR_INVALID, "residual_norm_grad: NULL pointer");
  if (workspace_bytes < opus_residual_norm_grad_workspace_bytes(&a))
    return set_error(OPUS_ERR_INVALID, "residual_norm_grad: workspace of %lld bytes, need %lld", (long long)workspace_bytes,
                     (long long)opus_residual_norm_grad_workspace_bytes(&a));
  if (!on(workspace, 256)) return set_error(OPUS_ERR_INVALID, "residual_norm_grad: workspace must be 256-byte aligned");
  const int xb = dtype_bytes(a.x_dtype), yb = dtype_bytes(a.y_dtype);
  if (a.h_stride < a.d || (a.y && a.y_stride < a.d) || (a.grad_n && a.grad_n_stride < a.d) ||
      (a.grad_h && a.grad_h_stride < a.d))
    return set_error(OPUS_ERR_INVALID, "residual_norm_grad: row stride < d");
  if (!on(a.h, xb) || !on(a.grad_h, xb) || !on(a.grad_x, xb) || !on(a.y, yb) || !on(a.grad_n, yb) ||
      !on(a.grad_y, yb) || !on(a.stats, 16))
    return set_error(OPUS_ERR_INVALID, "residual_norm_grad: a pointer is not aligned to its elements");
  const int V = 16 / xb;
  const bool vec = norm_params_aligned(&a) && a.d % V == 0 && a.h_stride % V == 0 && on(a.h, 16) && on(a.grad_x, 16) && on(a.grad_y, V * yb) &&
                   (!a.y || (a.y_stride % V == 0 && on(a.y, V * yb))) &&
                   (!a.grad_n || (a.grad_n_stride % V == 0 && on(a.grad_n, V * yb))) &&
                   (!a.grad_h || (a.grad_h_stride % V == 0 && on(a.grad_h, 16)));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const ColumnOutputs out{{outs[0], outs[1], outs[2], outs[3], outs[4]}, {types[0], types[1], types[2], types[3], types[4]}};
  if (a.x_dtype == OPUS_DTYPE_F32) {
    if (a.y_dtype == OPUS_DTYPE_F32) return residual_norm_grad_f32(a, vec, wanted, out, ws, st);
    if (a.y_dtype == OPUS_DTYPE_F16) return residual_norm_grad_f32_f16(a, vec, wanted, out, ws, st);
    return residual_norm_grad_f32_bf16(a, vec, wanted, out, ws, st);
  }
  if (a.x_dtype == OPUS_DTYPE_F16) return residual_norm_grad_f16(a, vec, wanted, out, ws, st);
  return residual_norm_grad_bf16(a, vec, wanted, out, ws, st);
}
