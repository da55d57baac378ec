// extern "C" entry points declared in include/mamba3_b200_lm.h: host-side
// validation, then one launch on the caller's stream.
#include <cstdint>

#include "m3_lm.cuh"

namespace {

bool dtype_ok(int32_t dt) { return dt == M3_F32 || dt == M3_BF16; }
bool aligned(const void *p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool dtype_aligned(const void *p, int32_t dt) { return aligned(p, dt == M3_BF16 ? 2 : 4); }

int check_device() {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) {
    cudaGetLastError();
    return M3_ERR_DEVICE;
  }
  return M3_OK;
}

// What both logit entry points ask of their inputs.
int check_logits(const m3_logits_args *a) {
  if (!a || !a->logits) return M3_ERR_NULL;
  if (!dtype_ok(a->dtype)) return M3_ERR_DTYPE;
  if (a->B < 0 || a->V <= 0 || a->V > (1 << 30) || a->T < 0 || a->ld < 0 || a->tokens_stride < 0 || a->bias_stride < 0 ||
      a->allowed_stride < 0)
    return M3_ERR_SHAPE;
  if (!dtype_aligned(a->logits, a->dtype) || !aligned(a->tokens, a->tokens_i64 ? 8 : 4) ||
      !aligned(a->lengths, a->lengths_i64 ? 8 : 4) || !aligned(a->prompt_lengths, a->prompt_i64 ? 8 : 4) ||
      !aligned(a->repetition, 4) || !aligned(a->presence, 4) || !aligned(a->frequency, 4) || !aligned(a->bias, 4) ||
      !aligned(a->allowed, 4))
    return M3_ERR_ALIGN;
  return M3_OK;
}

int launch_status(cudaError_t e) { return e == cudaSuccess ? M3_OK : M3_ERR_LAUNCH; }

}  // namespace

extern "C" {

int m3_linear_w4(const m3_w4_args *a, m3_stream_t stream) {
  if (!a || !a->x || !a->codes || !a->scales || !a->y) return M3_ERR_NULL;
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->s_dtype) || !dtype_ok(a->y_dtype)) return M3_ERR_DTYPE;
  if (a->group != 32 && a->group != 64 && a->group != 128) return M3_ERR_SHAPE;
  if (a->M < 0 || a->N <= 0 || a->K <= 0 || a->ldx < 0 || a->ldy < a->N) return M3_ERR_SHAPE;
  const int64_t groups = ((int64_t)a->K + a->group - 1) / a->group;
  if (a->scale_stride < groups || (a->zeros && a->zero_stride < groups)) return M3_ERR_SHAPE;
  // the kernels' 32-bit byte offsets into codes, scales and zeros
  const int64_t rows = ((int64_t)a->N + M3_W4_ROWS - 1) / M3_W4_ROWS;
  const int64_t tiles = ((int64_t)a->K + M3_W4_TILE - 1) / M3_W4_TILE;
  const int64_t most = (int64_t)1 << 32;
  if (rows * tiles > most / 1024 || (a->N - 1) > (most / 4 - groups) / a->scale_stride ||
      (a->zeros && (a->N - 1) > (most - groups) / a->zero_stride))
    return M3_ERR_SHAPE;
  if (!aligned(a->codes, 16)) return M3_ERR_ALIGN;
  if (!dtype_aligned(a->x, a->x_dtype) || !dtype_aligned(a->scales, a->s_dtype) || !dtype_aligned(a->y, a->y_dtype))
    return M3_ERR_ALIGN;
  if (a->M == 0) return M3_OK;
  const int st = check_device();
  if (st != M3_OK) return st;
  return launch_status(m3::launch_linear_w4(*a, reinterpret_cast<cudaStream_t>(stream)));
}

int m3_process_logits(const m3_logits_args *a, m3_stream_t stream) {
  int st = check_logits(a);
  if (st != M3_OK) return st;
  if (!a->out) return M3_ERR_NULL;
  if (!dtype_ok(a->out_dtype)) return M3_ERR_DTYPE;
  if (a->out_ld < a->V) return M3_ERR_SHAPE;
  if (!dtype_aligned(a->out, a->out_dtype)) return M3_ERR_ALIGN;
  if (a->B == 0) return M3_OK;
  if ((st = check_device()) != M3_OK) return st;
  return launch_status(m3::launch_process_logits(*a, reinterpret_cast<cudaStream_t>(stream)));
}

int m3_next_tokens(const m3_logits_args *a, m3_stream_t stream) {
  int st = check_logits(a);
  if (st != M3_OK) return st;
  if (!a->ids || !a->logprobs || (a->sample && !a->seeds)) return M3_ERR_NULL;
  if (!aligned(a->ids, 8) || !aligned(a->logprobs, 4) || !aligned(a->temperature, 4) || !aligned(a->seeds, 8) ||
      !aligned(a->positions, 8))
    return M3_ERR_ALIGN;
  if (a->B == 0) return M3_OK;
  if ((st = check_device()) != M3_OK) return st;
  return launch_status(m3::launch_next_tokens(*a, reinterpret_cast<cudaStream_t>(stream)));
}

}  // extern "C"
