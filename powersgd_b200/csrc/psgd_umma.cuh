// Matrix products of 16-bit operands on the tensor cores (tcgen05, kind::f16), with accumulators and one operand in
// tensor memory: what the attention kernels share.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "psgd_async.cuh"
#include "psgd_pairs.cuh"

// A panel is 64 or 128 rows of 64 elements of 16 bits, 128 bytes per row, as a TMA load with the 128-byte swizzle leaves it (eight rows, 1 KiB,
// are one swizzle atom). Wider tiles are several panels, one behind another.
constexpr int UMMA_ROWS = 128;
constexpr int UMMA_PANEL = UMMA_ROWS * 128;   // bytes

// Shared-memory descriptor of such a tile, 128-byte swizzle. Read along its rows (K-major): atoms follow each other along M or N
// every 1024 bytes; a step of 16 along K is 32 bytes further. Read across (MN-major: the rows are K): atoms follow each other along K every
// 1024 bytes, along N every `panel` bytes; a step of 16 along K is 2048 bytes further.
__device__ __forceinline__ uint64_t umma_tile(uint32_t saddr, uint32_t panel) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor: D float32, A and B of one type (0 float16, 1 bfloat16), M = 128.
__host__ __device__ constexpr uint32_t umma_shape(int type, bool b_across, int n) {
  return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) | ((b_across ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(UMMA_ROWS >> 4) << 24);
}

// A value that all lanes of the warp have, said so that the compiler knows: what follows from it lives in uniform registers, and a branch on it
// does not part the warp.
template <typename T>
__device__ __forceinline__ T warp_uniform(T x) { return __shfl_sync(0xffffffffu, x, 0); }

// The products are issued by a whole warp in step, one elected lane of it doing so: descriptors stay in uniform registers, where the
// instruction wants them. (Issued from a branch that one lane takes, a product took 80 cycles to issue and 32 to execute.)
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool accumulate) {   // A in tensor memory, K-major
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(shape), "r"((uint32_t)accumulate)
      : "memory");
}
// Arrives on `bar` when the products issued by this warp so far are complete.
__device__ __forceinline__ void umma_arrive(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(psgd_smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void umma_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void umma_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// D[128 x n] = A B^T over 16 `steps` elements: 128 rows of A, n of B (a panel of B has B_ROWS), both in shared memory.
template <int MOST_STEPS, int B_ROWS>
__device__ __forceinline__ void umma_rows_by_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, int steps) {
  const uint64_t ta = umma_tile(a, UMMA_PANEL), tb = umma_tile(b, B_ROWS * 128);
#pragma unroll
  for (int s = 0; s < MOST_STEPS; ++s) {
    if (s >= steps) break;   // (addresses are below 256 KiB: nothing is carried out of their field)
    umma_ss(d, ta + (((s >> 2) * UMMA_PANEL + (s & 3) * 32) >> 4), tb + (((s >> 2) * B_ROWS * 128 + (s & 3) * 32) >> 4), shape, s > 0);
  }
}
// D[128 x n] (+)= A B over rows [16 FROM, 16 TO) of B: A in tensor memory, eight columns for every 16 of K and GAP columns between those for
// every 32; B_ROWS rows of B are K.
template <int FROM, int TO, int B_ROWS, int GAP = 0>
__device__ __forceinline__ void umma_weights_by_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, bool accumulate) {
  const uint64_t tb = umma_tile(b, B_ROWS * 128);
#pragma unroll
  for (int s = FROM; s < TO; ++s) umma_ts(d, a + s * 8 + s / 2 * GAP, tb + (s * 2048 >> 4), shape, accumulate || s > 0);
}
// D[128 x n] += A B^T over 16 elements. Both lie without a swizzle: elements 0 to 7 of all rows, 16 bytes to a row, then elements 8 to 15.
template <int A_ROWS, int B_ROWS>
__device__ __forceinline__ void umma_add_columns(uint32_t d, uint32_t a, uint32_t b, uint32_t shape) {
  // (eight rows, 128 bytes, are one unit; the next rows' follows it, the next elements' is a whole column of them further)
  auto tile = [](uint32_t saddr, int rows) { return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(rows * 16 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46); };
  umma_ss(d, tile(a, A_ROWS), tile(b, B_ROWS), shape, true);
}

// 32 columns of the 32 lanes of this warp. A wait must follow before the registers are used.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float* f) {
  uint32_t* r = reinterpret_cast<uint32_t*>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
// Waits for the loads of this thread; `f` is what they fill (said to the compiler, which must not use it earlier).
template <int N>
__device__ __forceinline__ void tmem_load_wait(float* f) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(f[i])::"memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
               "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_alloc(uint32_t* at, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(psgd_smem_u32(at)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns) : "memory");
}

__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// Loads one box of a three-dimensional tensor.
__device__ __forceinline__ void tma_load_box3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map),
               "r"(psgd_smem_u32(bar)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// Two floats as a pair of 16-bit numbers, the first one in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
