// C ABI of the training step's operators around the memory layer: argument
// checks for norm.cu, loss.cu and orth.cu.
#include <math.h>
#include <stdint.h>

#include "loss.cuh"
#include "norm.cuh"
#include "orth.cuh"

namespace {

using namespace ml;

bool dtype_ok(int t) { return t == MEMLAYER_F32 || t == MEMLAYER_F16 || t == MEMLAYER_BF16; }

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

// A [rows, width] input: present, aligned to its element, rows that do not overlap.
int check_rows(const void* p, int64_t rows, int64_t stride, int64_t width, size_t esize) {
  if (rows == 0) return MEMLAYER_OK;
  if (!p || !aligned(p, esize)) return MEMLAYER_ERR_BAD_POINTER;
  if (stride < width || stride > (1ll << 40)) return MEMLAYER_ERR_BAD_SHAPE;
  return MEMLAYER_OK;
}

int check_norm(const memlayer_norm_config* c) {
  if (!c) return MEMLAYER_ERR_BAD_POINTER;
  if (c->rows < 0 || c->rows > (1ll << 40) || c->d_model < 1 || !(c->epsilon > 0.f) || !isfinite(c->epsilon))
    return MEMLAYER_ERR_BAD_SHAPE;
  if (!dtype_ok(c->dtype) || c->d_model > kNormMaxWidth) return MEMLAYER_ERR_UNSUPPORTED;
  return MEMLAYER_OK;
}

int check_loss(const memlayer_loss_config* c) {
  if (!c) return MEMLAYER_ERR_BAD_POINTER;
  if (c->tokens < 0 || c->tokens >= (1ll << 31) || c->d_model < 1 || c->vocab_size < 1) return MEMLAYER_ERR_BAD_SHAPE;
  // the last column tile's columns stay below 2^31
  if (!dtype_ok(c->dtype) || c->d_model > 65536 || c->vocab_size > 0x7FFFFF00) return MEMLAYER_ERR_UNSUPPORTED;
  return MEMLAYER_OK;
}

int check_orth(const memlayer_orth_config* c) {
  if (!c) return MEMLAYER_ERR_BAD_POINTER;
  if (c->batch < 0 || c->batch > 65535 || c->rows < 1 || c->cols < 1 || c->steps < 1 || !(c->epsilon >= 0.f) ||
      !isfinite(c->epsilon))
    return MEMLAYER_ERR_BAD_SHAPE;
  if (!dtype_ok(c->dtype) || c->rows > 32768 || c->cols > 32768 || c->steps > 64 || !orth_coefficients_ok(*c))
    return MEMLAYER_ERR_UNSUPPORTED;
  return MEMLAYER_OK;
}

size_t esize(int dtype) { return dtype == MEMLAYER_F32 ? 4 : 2; }

int check_loss_args(const memlayer_loss_config* c, const memlayer_loss_args* a) {
  if (!a) return MEMLAYER_ERR_BAD_POINTER;
  int st = check_rows(a->h, c->tokens, a->h_stride, c->d_model, esize(c->dtype));
  if (st) return st;
  if ((st = check_rows(a->weight, c->vocab_size, a->weight_stride, c->d_model, esize(c->dtype)))) return st;
  if (c->tokens > 0 && (!a->targets || !aligned(a->targets, 4))) return MEMLAYER_ERR_BAD_POINTER;
  return MEMLAYER_OK;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  return !ws || have < need || !aligned(ws, 256) ? MEMLAYER_ERR_WORKSPACE : MEMLAYER_OK;
}

int cuda_status(cudaError_t e) { return e == cudaSuccess ? MEMLAYER_OK : MEMLAYER_ERR_CUDA; }

}  // namespace

extern "C" {

int32_t memlayer_layer_norm(const memlayer_norm_config* cfg, const memlayer_norm_args* a, void* stream) {
  int st = check_norm(cfg);
  if (st) return st;
  if (!a) return MEMLAYER_ERR_BAD_POINTER;
  const size_t es = esize(cfg->dtype);
  if ((st = check_rows(a->x, cfg->rows, a->x_stride, cfg->d_model, es))) return st;
  if (a->residual && (st = check_rows(a->residual, cfg->rows, a->residual_stride, cfg->d_model, es))) return st;
  if (!a->scale || !a->bias || !aligned(a->scale, 4) || !aligned(a->bias, 4)) return MEMLAYER_ERR_BAD_POINTER;
  if (cfg->rows > 0 && (!a->y || !aligned(a->y, es) || !aligned(a->sum, es))) return MEMLAYER_ERR_BAD_POINTER;
  return cuda_status(launch_layer_norm(*cfg, *a, (cudaStream_t)stream));
}

int32_t memlayer_layer_norm_backward_workspace_size(const memlayer_norm_config* cfg, size_t* bytes) {
  const int st = check_norm(cfg);
  if (st) return st;
  if (!bytes) return MEMLAYER_ERR_BAD_POINTER;
  // the head holds the status word
  *bytes = 512 + (size_t)norm_backward_blocks(cfg->rows, cfg->d_model, cfg->dtype) * 2 * cfg->d_model * sizeof(float);
  return MEMLAYER_OK;
}

int32_t memlayer_layer_norm_backward(const memlayer_norm_config* cfg, const memlayer_norm_grads* g, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  size_t need = 0;
  int st = memlayer_layer_norm_backward_workspace_size(cfg, &need);
  if (st) return st;
  if (!g) return MEMLAYER_ERR_BAD_POINTER;
  const size_t es = esize(cfg->dtype);
  if ((st = check_rows(g->dy, cfg->rows, g->dy_stride, cfg->d_model, es))) return st;
  if ((st = check_rows(g->x, cfg->rows, g->x_stride, cfg->d_model, es))) return st;
  if (g->dresidual && (st = check_rows(g->dresidual, cfg->rows, g->dresidual_stride, cfg->d_model, es))) return st;
  if (!g->scale || !g->dscale || !g->dbias || !aligned(g->scale, 4) || !aligned(g->dscale, 4) ||
      !aligned(g->dbias, 4))
    return MEMLAYER_ERR_BAD_POINTER;
  if (cfg->rows > 0 && (!g->dx || !aligned(g->dx, es))) return MEMLAYER_ERR_BAD_POINTER;
  if ((st = check_workspace(workspace, workspace_bytes, need))) return st;
  char* ws = (char*)workspace;
  return cuda_status(launch_layer_norm_backward(*cfg, *g, (float*)(ws + 512), (int*)(ws + 256), (cudaStream_t)stream));
}

int32_t memlayer_cross_entropy_workspace_size(const memlayer_loss_config* cfg, int32_t backward, size_t* bytes) {
  const int st = check_loss(cfg);
  if (st) return st;
  if (!bytes) return MEMLAYER_ERR_BAD_POINTER;
  return loss_workspace(*cfg, backward != 0, bytes) ? MEMLAYER_OK : MEMLAYER_ERR_UNSUPPORTED;
}

int32_t memlayer_cross_entropy(const memlayer_loss_config* cfg, const memlayer_loss_args* a, void* workspace,
                               size_t workspace_bytes, void* stream) {
  size_t need = 0;
  int st = memlayer_cross_entropy_workspace_size(cfg, 0, &need);
  if (st) return st;
  if ((st = check_loss_args(cfg, a))) return st;
  if (cfg->tokens > 0 && (!a->loss || !a->lse || !aligned(a->loss, 4) || !aligned(a->lse, 4)))
    return MEMLAYER_ERR_BAD_POINTER;
  if ((st = check_workspace(workspace, workspace_bytes, need))) return st;
  return cuda_status(launch_loss_forward(*cfg, *a, (char*)workspace, (cudaStream_t)stream));
}

int32_t memlayer_cross_entropy_backward(const memlayer_loss_config* cfg, const memlayer_loss_args* a,
                                        const memlayer_loss_grads* g, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  size_t need = 0;
  int st = memlayer_cross_entropy_workspace_size(cfg, 1, &need);
  if (st) return st;
  if ((st = check_loss_args(cfg, a))) return st;
  if (!g || !g->dweight || !aligned(g->dweight, esize(cfg->dtype))) return MEMLAYER_ERR_BAD_POINTER;
  if (cfg->tokens > 0 && (!g->lse || !g->dloss || !g->dh || !aligned(g->lse, 4) || !aligned(g->dloss, 4) ||
                          !aligned(g->dlse, 4) || !aligned(g->dh, esize(cfg->dtype))))
    return MEMLAYER_ERR_BAD_POINTER;
  if ((st = check_workspace(workspace, workspace_bytes, need))) return st;
  return cuda_status(launch_loss_backward(*cfg, *a, *g, (char*)workspace, (cudaStream_t)stream));
}

int32_t memlayer_train_status(const void* workspace, int32_t* code, void* stream) {
  if (!workspace || !code) return MEMLAYER_ERR_BAD_POINTER;
  int v = 0;
  if (cudaMemcpyAsync(&v, (const char*)workspace + 256, sizeof(int), cudaMemcpyDeviceToHost, (cudaStream_t)stream) !=
          cudaSuccess ||
      cudaStreamSynchronize((cudaStream_t)stream) != cudaSuccess)
    return MEMLAYER_ERR_CUDA;
  *code = v;
  return MEMLAYER_OK;
}

int32_t memlayer_orthogonalize_workspace_size(const memlayer_orth_config* cfg, size_t* bytes) {
  const int st = check_orth(cfg);
  if (st) return st;
  if (!bytes) return MEMLAYER_ERR_BAD_POINTER;
  return orth_workspace(*cfg, bytes) ? MEMLAYER_OK : MEMLAYER_ERR_UNSUPPORTED;
}

int32_t memlayer_orthogonalize(const memlayer_orth_config* cfg, const void* update, void* out, void* workspace,
                               size_t workspace_bytes, void* stream) {
  size_t need = 0;
  int st = memlayer_orthogonalize_workspace_size(cfg, &need);
  if (st) return st;
  const size_t es = esize(cfg->dtype);
  if (cfg->batch > 0 && (!update || !out || !aligned(update, es) || !aligned(out, es)))
    return MEMLAYER_ERR_BAD_POINTER;
  if ((st = check_workspace(workspace, workspace_bytes, need))) return st;
  return cuda_status(launch_orthogonalize(*cfg, update, out, (char*)workspace, (cudaStream_t)stream));
}

}  // extern "C"
