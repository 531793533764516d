// The rotation of heads for bfloat16.
#include "rotary.cuh"

int psgd_rotate_bfloat16(const PsgdRotate* call, bool gradient, cudaStream_t stream) { return rt_call<__nv_bfloat16>(call, gradient, stream); }
