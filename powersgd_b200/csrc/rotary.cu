// Entry points of the rotation of heads, and its kernels for float32 (rotary.cuh).
#include "rotary.cuh"

int psgd_rotate_float32(const PsgdRotate* call, bool gradient, cudaStream_t stream) { return rt_call<float>(call, gradient, stream); }

static int rotate(const PsgdRotate* call, bool gradient, cudaStream_t stream) {
  if (call->rows == 0) return 0;
  if (call->heads + call->keys > RT_MOST_HEADS || call->size < 8 || call->size > RT_MOST_SIZE || call->size % 8 || call->rotated < 0 || call->rotated > call->size || call->rotated % 8) {
    psgd_set_error("psgd_rotate: %d heads of %d of which %d are turned", call->heads + call->keys, call->size, call->rotated);
    return PSGD_BAD_ARGUMENT;
  }
  if (call->type == 0) return psgd_rotate_float32(call, gradient, stream);
  if (call->type == 1) return psgd_rotate_bfloat16(call, gradient, stream);
  return psgd_rotate_float16(call, gradient, stream);
}

// Numbers of 64 bits, scratch for the gradients of weights.
PSGD_API long long psgd_rotate_parts(int size) { return (long long)RT_PART_BLOCKS * 2 * size; }

// `call`: host memory, read before the call returns. Rows that belong to no sequence give zeros.
PSGD_API int psgd_rotate(const PsgdRotate* call, cudaStream_t stream) { return rotate(call, false, stream); }

// The gradients of x (all of it, values included) and of the weights.
PSGD_API int psgd_rotate_grad(const PsgdRotate* call, cudaStream_t stream) { return rotate(call, true, stream); }
