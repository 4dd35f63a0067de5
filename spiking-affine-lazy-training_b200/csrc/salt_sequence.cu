// C ABI of the sequence operators: argument checks, then the launches of seq_*.cu.
#include <string>

#include "salt_host.h"
#include "sequence.cuh"

namespace salt {
namespace {

constexpr int32_t kMostLen = 1 << 30;
constexpr int32_t kMostDim = 1 << 24;

// Whether no two of rows * len runs of `dim` elements, at b * batch + t * token, share an element.
bool apart(int64_t batch, int64_t token, int32_t rows, int32_t len, int32_t dim) {
  if (rows < 1 || len < 1) return true;
  if ((len > 1 && token < dim) || (rows > 1 && batch < dim)) return false;
  if (len == 1 || rows == 1) return true;
  using wide = __int128;
  // one axis lies within a step of the other, either way around
  if (batch >= (wide)(len - 1) * token + dim || token >= (wide)(rows - 1) * batch + dim) return true;
  // else a step of one axis must not meet any of the other: only the two around it can
  const bool few = rows < len;
  const int64_t outer = few ? batch : token, inner = few ? token : batch;
  const int32_t steps = few ? rows : len, most = few ? len : rows;
  for (int32_t i = 1; i < steps; ++i) {
    const wide at = (wide)i * outer, j = at / inner;
    if ((j < most && at - j * inner < dim) || (j + 1 < most && (j + 1) * inner - at < dim))
      return false;
  }
  return true;
}

// The first failed check of a call; `ok` stays true while all hold.
struct Checks {
  const char* who;
  std::string why;
  explicit Checks(const char* w) : who(w) {}
  bool ok() const { return why.empty(); }
  void need(bool cond, const char* text) {
    if (!cond && ok()) why = std::string(who) + ": " + text;
  }
  void type(int32_t t) {
    need(t == SALT_F32 || t == SALT_F16 || t == SALT_BF16, "type must be SALT_F32, F16 or BF16");
  }
  // `other` holds the activations' type or float32
  void wide(int32_t other, int32_t t, const char* text) {
    need(other == t || other == SALT_F32, text);
  }
  void input(const void* p, bool used, const char* text) { need(!used || p, text); }
  // rows of an array: strides are not negative, and rows that are written do not overlap
  void strides(int64_t batch, int64_t token, const char* text) {
    need(batch >= 0 && token >= 0, text);
  }
  void written(int64_t batch, int64_t token, int32_t rows, int32_t len, int32_t dim,
               const char* text) {
    if (ok()) need(batch >= 0 && token >= 0 && apart(batch, token, rows, len, dim), text);
  }
  salt_status status() const { return host_fail(SALT_BAD_ARG, why); }
};

salt_status launched(cudaError_t e, int launches, const char* who) {
  host_launched(launches);
  if (e != cudaSuccess)
    return host_fail(SALT_CUDA_ERROR, std::string(who) + ": " + cudaGetErrorString(e));
  return SALT_OK;
}

salt_status room(const char* who, const void* ws, size_t have, size_t need) {
  if (need == 0) return SALT_OK;
  if (!ws || have < need)
    return host_fail(SALT_WORKSPACE_TOO_SMALL, std::string(who) + ": workspace needs " +
                                                   std::to_string(need) + " bytes, got " +
                                                   std::to_string(ws ? have : 0));
  if (reinterpret_cast<uintptr_t>(ws) % 256)
    return host_fail(SALT_BAD_ARG, std::string(who) + ": workspace is not 256-byte aligned");
  return SALT_OK;
}

void shape(Checks& c, int32_t batch, int32_t len, int32_t dim) {
  c.need(batch >= 0, "batch is negative");
  c.need(len >= 0 && len <= kMostLen, "len must lie in [0, 2^30]");
  c.need(dim >= 1 && dim <= kMostDim, "dim must lie in [1, 2^24]");
  // a launch has at most one block for 8 tokens of 32 channels (and one for a shorter rest)
  c.need((int64_t)batch * (len / 8 + 1) <= (int64_t)0x7fffffff / (dim / 16 + 1),
         "batch * len * dim is too large for one launch");
}

Checks check(const salt_rms_norm_args* a) {
  Checks c("salt_rms_norm");
  c.need(a, "args is NULL");
  if (!c.ok()) return c;
  c.type(a->type);
  c.wide(a->residual_type, a->type, "residual_type must be type or SALT_F32");
  c.wide(a->weight_type, a->type, "weight_type must be type or SALT_F32");
  c.need(a->rows >= 0, "rows is negative");
  c.need(a->dim >= 1 && a->dim <= 16384, "dim must lie in [1, 16384]");
  c.need(a->eps >= 0.f, "eps must not be negative");
  c.need(!a->scale || a->group == 0 || a->group == 32 || a->group == 64 || a->group == 128 ||
             a->group == 256,
         "group must be 0, 32, 64, 128 or 256");
  const bool used = a->rows > 0;
  c.input(a->x, used, "x is NULL");
  c.input(a->weight, used, "weight is NULL");
  c.input(a->out, used, "out is NULL");
  c.strides(a->x_stride, a->residual_stride, "a stride is negative");
  c.written(0, a->out_stride, 1, a->rows, a->dim, "out_stride must be at least dim");
  if (a->residual_out)
    c.written(0, a->residual_out_stride, 1, a->rows, a->dim,
              "residual_out_stride must be at least dim");
  return c;
}

Checks check(const salt_rms_norm_backward_args* a) {
  Checks c("salt_rms_norm_backward");
  c.need(a, "args is NULL");
  if (!c.ok()) return c;
  c.type(a->type);
  c.wide(a->residual_type, a->type, "residual_type must be type or SALT_F32");
  c.wide(a->weight_type, a->type, "weight_type must be type or SALT_F32");
  c.need(a->rows >= 0, "rows is negative");
  c.need(a->dim >= 1 && a->dim <= 16384, "dim must lie in [1, 16384]");
  const bool used = a->rows > 0;
  c.input(a->dy, used, "dy is NULL");
  c.input(a->x, used, "x is NULL");
  c.input(a->weight, true, "weight is NULL");  // without rows, too, a block loads it
  c.input(a->rstd, used, "rstd is NULL");
  c.input(a->dx, used, "dx is NULL");
  c.strides(a->dy_stride, a->x_stride, "a stride is negative");
  c.strides(a->dresidual_stride, 0, "a stride is negative");
  c.written(0, a->dx_stride, 1, a->rows, a->dim, "dx_stride must be at least dim");
  return c;
}

template <class A>
void conv_common(Checks& c, const A* a) {
  c.type(a->type);
  c.wide(a->weight_type, a->type, "weight_type must be type or SALT_F32");
  c.need(a->width >= 1 && a->width <= 8, "width must lie in [1, 8]");
}

Checks check(const salt_causal_conv_args* a) {
  Checks c("salt_causal_conv");
  c.need(a, "args is NULL");
  if (!c.ok()) return c;
  conv_common(c, a);
  shape(c, a->batch, a->len, a->dim);
  // a thread takes one channel through 32 tokens at most there, and counts its row's in 32 bits
  c.need((int64_t)a->dim * (((int64_t)a->len + 31) / 32) <= (int64_t)UINT32_MAX,
         "len * dim is too large for one launch");
  const bool used = a->batch > 0 && a->len > 0;
  c.input(a->x, used, "x is NULL");
  c.input(a->weight, used, "weight is NULL");
  c.input(a->out, used, "out is NULL");
  c.strides(a->x_batch_stride, a->x_stride, "a stride is negative");
  c.written(a->out_batch_stride, a->out_stride, a->batch, a->len, a->dim,
            "out's strides let its rows overlap");
  return c;
}

Checks check(const salt_causal_conv_step_args* a) {
  Checks c("salt_causal_conv_step");
  c.need(a, "args is NULL");
  if (!c.ok()) return c;
  conv_common(c, a);
  shape(c, a->batch, 1, a->dim);
  c.need(a->n_slots >= 0, "n_slots is negative");
  c.need(a->slots || a->batch <= a->n_slots, "without slots, batch must not exceed n_slots");
  const bool used = a->batch > 0;
  c.input(a->x, used, "x is NULL");
  c.input(a->weight, used, "weight is NULL");
  c.input(a->out, used, "out is NULL");
  c.input(a->state, used && a->width > 1 && a->n_slots > 0, "state is NULL");
  c.strides(a->x_stride, 0, "a stride is negative");
  c.written(0, a->out_stride, 1, a->batch, a->dim, "out_stride must be at least dim");
  return c;
}

Checks check(const salt_causal_conv_backward_args* a) {
  Checks c("salt_causal_conv_backward");
  c.need(a, "args is NULL");
  if (!c.ok()) return c;
  conv_common(c, a);
  shape(c, a->batch, a->len, a->dim);
  const bool used = a->batch > 0 && a->len > 0;
  c.input(a->dy, used, "dy is NULL");
  c.input(a->x, used, "x is NULL");
  c.input(a->weight, a->batch > 0, "weight is NULL");  // rows without tokens load it, too
  c.input(a->dx, used, "dx is NULL");
  c.input(a->dweight, true, "dweight is NULL");
  c.strides(a->x_batch_stride, a->x_stride, "a stride is negative");
  c.strides(a->dy_batch_stride, a->dy_stride, "a stride is negative");
  c.written(a->dx_batch_stride, a->dx_stride, a->batch, a->len, a->dim,
            "dx's strides let its rows overlap");
  return c;
}

template <class A>
void scan_common(Checks& c, const A* a, int32_t len) {
  c.type(a->type);
  shape(c, a->batch, len, a->dim);
  c.need(a->state >= 1 && a->state <= 64, "state must lie in [1, 64]");
  c.need(a->groups >= 1 && a->dim % (a->groups < 1 ? 1 : a->groups) == 0,
         "groups must divide dim");
  // a group has blocks of its own, and dB and dC a value for each of its states
  c.need((int64_t)a->batch * (len / 8 + 1) <= (int64_t)0x7fffffff / (a->groups < 1 ? 1 : a->groups),
         "batch * len * groups is too large for one launch");
  const bool used = a->batch > 0 && len > 0;
  c.input(a->x, used, "x is NULL");
  c.input(a->delta, used, "delta is NULL");
  c.input(a->B, used, "B is NULL");
  c.input(a->C, used, "C is NULL");
  c.input(a->A, a->batch > 0, "A is NULL");  // rows without tokens load it, too
  c.strides(a->x_stride, a->delta_stride, "a stride is negative");
  c.strides(a->B_stride, a->C_stride, "a stride is negative");
  c.strides(a->z_stride, 0, "a stride is negative");
}

template <class A>
void scan_batch_strides(Checks& c, const A* a) {
  c.strides(a->x_batch_stride, a->delta_batch_stride, "a stride is negative");
  c.strides(a->B_batch_stride, a->C_batch_stride, "a stride is negative");
  c.strides(a->z_batch_stride, 0, "a stride is negative");
}

Checks check(const salt_selective_scan_args* a) {
  Checks c("salt_selective_scan");
  c.need(a, "args is NULL");
  if (!c.ok()) return c;
  scan_common(c, a, a->len);
  scan_batch_strides(c, a);
  c.input(a->out, a->batch > 0 && a->len > 0, "out is NULL");
  c.written(a->out_batch_stride, a->out_stride, a->batch, a->len, a->dim,
            "out's strides let its rows overlap");
  return c;
}

Checks check(const salt_selective_scan_step_args* a) {
  Checks c("salt_selective_scan_step");
  c.need(a, "args is NULL");
  if (!c.ok()) return c;
  scan_common(c, a, 1);
  c.need(a->n_slots >= 0, "n_slots is negative");
  c.need(a->slots || a->batch <= a->n_slots, "without slots, batch must not exceed n_slots");
  c.input(a->pool, a->batch > 0 && a->n_slots > 0, "pool is NULL");
  c.input(a->out, a->batch > 0, "out is NULL");
  c.written(0, a->out_stride, 1, a->batch, a->dim, "out_stride must be at least dim");
  return c;
}

Checks check(const salt_selective_scan_backward_args* a) {
  Checks c("salt_selective_scan_backward");
  c.need(a, "args is NULL");
  if (!c.ok()) return c;
  scan_common(c, a, a->len);
  scan_batch_strides(c, a);
  // the kernel that writes dB and dC counts a token's values of both in 32 bits
  c.need((int64_t)2 * a->state * a->groups <= INT32_MAX, "groups * state is too large");
  const bool used = a->batch > 0 && a->len > 0;
  c.input(a->dy, used, "dy is NULL");
  c.input(a->checkpoints, used, "checkpoints is NULL");
  c.input(a->dx, used, "dx is NULL");
  c.input(a->ddelta, used, "ddelta is NULL");
  c.input(a->dB, used, "dB is NULL");
  c.input(a->dC, used, "dC is NULL");
  c.input(a->dA, true, "dA is NULL");
  c.need(!used || (a->z == nullptr) == (a->dz == nullptr), "dz is needed exactly where z is given");
  c.strides(a->dy_batch_stride, a->dy_stride, "a stride is negative");
  const char* text = "a gradient's strides let its rows overlap";
  c.written(a->dx_batch_stride, a->dx_stride, a->batch, a->len, a->dim, text);
  c.written(a->ddelta_batch_stride, a->ddelta_stride, a->batch, a->len, a->dim, text);
  if (a->dz) c.written(a->dz_batch_stride, a->dz_stride, a->batch, a->len, a->dim, text);
  return c;
}

}  // namespace
}  // namespace salt

using namespace salt;

extern "C" {

salt_status salt_rms_norm(const salt_rms_norm_args* args, void* stream) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  int n = 0;
  const cudaError_t e = rms_norm_launch(*args, (cudaStream_t)stream, &n);
  return launched(e, n, c.who);
}

salt_status salt_rms_norm_backward_workspace_size(const salt_rms_norm_backward_args* args,
                                                  size_t* bytes) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  if (!bytes) return host_fail(SALT_BAD_ARG, "bytes is NULL");
  *bytes = rms_norm_backward_bytes(*args);
  return SALT_OK;
}

salt_status salt_rms_norm_backward(const salt_rms_norm_backward_args* args, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  const salt_status s = room(c.who, workspace, workspace_bytes, rms_norm_backward_bytes(*args));
  if (s) return s;
  int n = 0;
  const cudaError_t e = rms_norm_backward_launch(*args, workspace, (cudaStream_t)stream, &n);
  return launched(e, n, c.who);
}

salt_status salt_causal_conv(const salt_causal_conv_args* args, void* stream) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  int n = 0;
  const cudaError_t e = causal_conv_launch(*args, (cudaStream_t)stream, &n);
  return launched(e, n, c.who);
}

salt_status salt_causal_conv_step(const salt_causal_conv_step_args* args, void* stream) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  int n = 0;
  const cudaError_t e = causal_conv_step_launch(*args, (cudaStream_t)stream, &n);
  return launched(e, n, c.who);
}

salt_status salt_causal_conv_backward_workspace_size(const salt_causal_conv_backward_args* args,
                                                     size_t* bytes) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  if (!bytes) return host_fail(SALT_BAD_ARG, "bytes is NULL");
  *bytes = causal_conv_backward_bytes(*args);
  return SALT_OK;
}

salt_status salt_causal_conv_backward(const salt_causal_conv_backward_args* args, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  const salt_status s = room(c.who, workspace, workspace_bytes, causal_conv_backward_bytes(*args));
  if (s) return s;
  int n = 0;
  const cudaError_t e = causal_conv_backward_launch(*args, workspace, (cudaStream_t)stream, &n);
  return launched(e, n, c.who);
}

salt_status salt_selective_scan_workspace_size(const salt_selective_scan_args* args,
                                               size_t* bytes) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  if (!bytes) return host_fail(SALT_BAD_ARG, "bytes is NULL");
  *bytes = selective_scan_bytes(*args);
  return SALT_OK;
}

salt_status salt_selective_scan(const salt_selective_scan_args* args, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  const salt_status s = room(c.who, workspace, workspace_bytes, selective_scan_bytes(*args));
  if (s) return s;
  int n = 0;
  const cudaError_t e = selective_scan_launch(*args, workspace, (cudaStream_t)stream, &n);
  return launched(e, n, c.who);
}

salt_status salt_selective_scan_step(const salt_selective_scan_step_args* args, void* stream) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  int n = 0;
  const cudaError_t e = selective_scan_step_launch(*args, (cudaStream_t)stream, &n);
  return launched(e, n, c.who);
}

salt_status salt_selective_scan_backward_workspace_size(
    const salt_selective_scan_backward_args* args, size_t* bytes) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  if (!bytes) return host_fail(SALT_BAD_ARG, "bytes is NULL");
  *bytes = selective_scan_backward_bytes(*args);
  return SALT_OK;
}

salt_status salt_selective_scan_backward(const salt_selective_scan_backward_args* args,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  const Checks c = check(args);
  if (!c.ok()) return c.status();
  const salt_status s =
      room(c.who, workspace, workspace_bytes, selective_scan_backward_bytes(*args));
  if (s) return s;
  int n = 0;
  const cudaError_t e = selective_scan_backward_launch(*args, workspace, (cudaStream_t)stream, &n);
  return launched(e, n, c.who);
}

}  // extern "C"
