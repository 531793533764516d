// The rotation of heads for float16.
#include "rotary.cuh"

int psgd_rotate_float16(const PsgdRotate* call, bool gradient, cudaStream_t stream) { return rt_call<__half>(call, gradient, stream); }
