// AdamW over a list of tensors in one launch, moments in 32 bits or in 8.
//
//   m <- b1 m + (1 - b1) g          v <- b2 v + (1 - b2) g^2          t <- t + 1
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in float32 whatever the type of p and g; p is rounded to its type once. A step moves 28 bytes per float32
// parameter (p, m, v in and out, g in), 16.1 with moments in 8 bits, and computes some tens of operations: the
// memory bounds it. A block takes 4096 elements of one tensor, found by a search in the list that the launch
// carries in its own arguments: nothing is uploaded, and a recorded launch keeps its list.
//
// The number of steps of a tensor, t, lives in device memory, so that a replayed graph counts on. Every block reads
// it; the last one to finish (a ticket) adds one to all of them.
//
// Moments in 8 bits: e4m3 values x = code * scale with one scale per 256 elements, largest / 448. Held are m and
// r = sqrt(v), whose range relative to the largest of a block, 1 : 2e5, is one of 1 : 5e10 in v. b2 = 0.999 moves r by
// 0.05 % of itself in a step where neighbouring codes lie 6 to 12 % apart: rounded to the nearest it would stand
// still, so a value is rounded up or down with the probabilities that keep its mean. What is not zero in r stays above
// zero: an element whose second moment rounded to nothing would next be divided by its newest gradient alone.
// The random bits are a hash of (seed, t, position), the finalizer of MurmurHash3 in three rounds: the same inputs
// give the same result. The update itself uses the moments before they are rounded.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "psgd_common.cuh"

namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_CHUNK = 4096;     // elements of a block
constexpr int AW_BLOCK = 256;      // elements that share a scale: one warp, eight per lane
constexpr int AW_GRID = 4 * 148;   // blocks that run at a time
constexpr float AW_E4M3_MAX = 448.f;

}  // namespace

// One tensor of a list, as the caller fills it in (ops/adamw.py).
typedef struct {
  void* p;
  const void* g;
  void* m;              // float32, or e4m3 codes
  void* v;              // float32, or e4m3 codes of the root
  float* m_scale;       // moments in 8 bits: a scale per 256 elements
  float* v_scale;
  float* step;
  long long n;
  uint32_t block0;      // first block of 256 of the tensor in the stream of random numbers
  uint32_t chunk_end;   // chunks of the list up to and with this tensor (filled in by the launch)
} PsgdAdamTensor;       // 72 bytes

namespace {

struct AwHyper {
  float lr;
  const float* lr_at;   // read instead of lr where it is not null
  float beta1, beta2, rest1, rest2, log_beta1, log_beta2, eps, decay;
  uint32_t seed;
  int* ticket;          // zero before the launch and after it
};

// A launch carries its list in the arguments (32 KiB at most): 40 tensors for short lists, whose launch is
// cheaper, 400 for long ones.
template <int MOST>
struct AwArgs {
  AwHyper h;
  int count;
  PsgdAdamTensor t[MOST];
};

template <typename T>
__device__ __forceinline__ void aw_load4(const T* p, float* f);
template <>
__device__ __forceinline__ void aw_load4<float>(const float* p, float* f) {
  const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
  f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
}
template <>
__device__ __forceinline__ void aw_load4<__nv_bfloat16>(const __nv_bfloat16* p, float* f) {
  const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
  f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xFFFF0000u);
  f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void aw_load4<__half>(const __half* p, float* f) {
  const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
__device__ __forceinline__ void aw_store4(float* p, const float* f) { __stcs(reinterpret_cast<float4*>(p), make_float4(f[0], f[1], f[2], f[3])); }
__device__ __forceinline__ void aw_store4(__nv_bfloat16* p, const float* f) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
  __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b)));
}
__device__ __forceinline__ void aw_store4(__half* p, const float* f) {
  const __half2 a = __floats2half2_rn(f[0], f[1]), b = __floats2half2_rn(f[2], f[3]);
  __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b)));
}
__device__ __forceinline__ float aw_get(const float* p) { return *p; }
__device__ __forceinline__ float aw_get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float aw_get(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void aw_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void aw_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void aw_put(__half* p, float v) { *p = __float2half_rn(v); }

// What a step multiplies with, from the number of steps.
struct AwFactors {
  float keep, size, inv_root2;   // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};
__device__ __forceinline__ AwFactors aw_factors(const AwHyper& h, float t) {
  const float lr = h.lr_at ? *h.lr_at : h.lr;
  AwFactors f;
  f.keep = 1.f - lr * h.decay;
  f.size = lr / -expm1f(t * h.log_beta1);
  f.inv_root2 = 1.f / sqrtf(-expm1f(t * h.log_beta2));
  return f;
}
// Products and sums are rounded one by one, without fused multiply-adds: moments are the same bits that elementwise operations give, and
// 8-bit codes that follow from them are too, in this step and in all later ones.
__device__ __forceinline__ void aw_moments(const AwHyper& h, float g, float& m, float& v) {
  m = __fadd_rn(__fmul_rn(m, h.beta1), __fmul_rn(g, h.rest1));
  v = __fadd_rn(__fmul_rn(v, h.beta2), __fmul_rn(__fmul_rn(g, g), h.rest2));
}
__device__ __forceinline__ float aw_update(const AwHyper& h, const AwFactors& f, float p, float m, float root) {
  return p * f.keep - f.size * __fdividef(m, root * f.inv_root2 + h.eps);   // (2 ulp; the update is small beside p)
}

// The tensor that holds chunk `c` of the list, the lo-th or a later one.
template <int MOST>
__device__ __forceinline__ int aw_find(const AwArgs<MOST>& a, uint32_t c, int lo) {
  int hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c < a.t[mid].chunk_end) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// The last block of the grid counts the step for every tensor: no block reads the number any more.
template <int MOST>
__device__ __forceinline__ void aw_count(const AwArgs<MOST>& a) {
  __shared__ int s_last;
  __syncthreads();
  if (threadIdx.x == 0) s_last = psgd_atom_add_acqrel_gpu(a.h.ticket, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  for (int i = threadIdx.x; i < a.count; i += AW_THREADS) *a.t[i].step += 1.f;
  if (threadIdx.x == 0) *a.h.ticket = 0;
}

// A block takes every gridDim.x-th chunk of the list: what it needs to know of a tensor it finds out once for most of its chunks.
#define AW_FOR_CHUNKS(a, t, first, f, steps)                                                             \
  int which = -1;                                                                                        \
  AwFactors f;                                                                                           \
  float steps = 0.f;                                                                                     \
  uint32_t first = 0, end = 0;                                                                           \
  const uint32_t chunks = a.t[a.count - 1].chunk_end;                                                    \
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {                                \
    if (chunk >= end) {                                                                                  \
      which = aw_find(a, chunk, which + 1);                                                              \
      first = which ? a.t[which - 1].chunk_end : 0;                                                      \
      end = a.t[which].chunk_end;                                                                        \
      const float now = *(volatile const float*)a.t[which].step + 1.f;                                   \
      if (now != steps) f = aw_factors(a.h, steps = now);                                                \
    }                                                                                                    \
    const PsgdAdamTensor& t = a.t[which];

template <typename T, int MOST>
__global__ void __launch_bounds__(AW_THREADS, 4) psgd_adamw_kernel(const __grid_constant__ AwArgs<MOST> a) {
  AW_FOR_CHUNKS(a, t, first, f, steps)
  const long long e0 = (long long)(chunk - first) * AW_CHUNK;
  const int left = (int)min((long long)AW_CHUNK, t.n - e0);
  T* p = (T*)t.p + e0;
  const T* g = (const T*)t.g + e0;
  float* m = (float*)t.m + e0;
  float* v = (float*)t.v + e0;
  const uintptr_t all = (uintptr_t)m | (uintptr_t)v;
  const bool wide = ((all & 15u) | (((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1))) == 0;
  if (wide && left == AW_CHUNK) {
    constexpr int U = 2;
#pragma unroll
    for (int half = 0; half < AW_CHUNK / (AW_THREADS * 4 * U); ++half) {
      float pp[U][4], gg[U][4], mm[U][4], vv[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (half * U + u) * AW_THREADS * 4 + threadIdx.x * 4;
        aw_load4(g + i, gg[u]);
        aw_load4((const float*)m + i, mm[u]);
        aw_load4((const float*)v + i, vv[u]);
        aw_load4((const T*)p + i, pp[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (half * U + u) * AW_THREADS * 4 + threadIdx.x * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          aw_moments(a.h, gg[u][j], mm[u][j], vv[u][j]);
          pp[u][j] = aw_update(a.h, f, pp[u][j], mm[u][j], sqrtf(vv[u][j]));
        }
        aw_store4(m + i, mm[u]);
        aw_store4(v + i, vv[u]);
        aw_store4(p + i, pp[u]);
      }
    }
  } else {   // the end of a tensor, or one that does not begin on a 16-byte boundary
    for (int i = threadIdx.x; i < left; i += AW_THREADS) {
      float mm = m[i], vv = v[i];
      aw_moments(a.h, aw_get(g + i), mm, vv);
      const float pp = aw_update(a.h, f, aw_get(p + i), mm, sqrtf(vv));
      m[i] = mm;
      v[i] = vv;
      aw_put(p + i, pp);
    }
  }
  }
  aw_count(a);
}

// ---- moments in 8 bits -------------------------------------------------------------------------
__device__ __forceinline__ uint32_t aw_mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x85EBCA6Bu;
  x ^= x >> 13;
  x *= 0xC2B2AE35u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ void aw_decode4(uint32_t codes, float scale, float* f) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * j)), __NV_E4M3);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
    f[2 * j] = __fmul_rn(x.x, scale);
    f[2 * j + 1] = __fmul_rn(x.y, scale);
  }
}

// The e4m3 value that `x * inv` is rounded to by 16 random bits. 20 bits of a float's mantissa lie below the three that stay: a random
// number of 20 bits (16, the middle of their step) is added and what lies below is cut. Steps below 2^-6 are those right above it, so
// that range is moved there and back. The conversion to e4m3 is exact but for its saturation. (Where the block holds what is
// no number its scale is none either, whatever the codes are.)
__device__ __forceinline__ float aw_round(float x, float inv, uint32_t random20, bool least) {
  const float y = __fmul_rn(fabsf(x), inv);
  const float shift = y < 0.015625f ? 0.015625f : 0.f;
  const float t = __fadd_rn(__uint_as_float((__float_as_uint(__fadd_rn(y, shift)) + random20) & 0xFFF00000u), -shift);
  if (least) return fmaxf(t, y > 0.f ? 0.001953125f : 0.f);
  return copysignf(t, x);
}
__device__ __forceinline__ uint32_t aw_encode4(const float* f) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// Scale of a block from the bits of its largest magnitude (as integers they order as the numbers do, and what is no number comes
// last). Below 2^-100 a block is taken for zeros: its scale and the reciprocal would leave the normal range.
__device__ __forceinline__ float aw_scale(uint32_t bits, float& inv) {
  const float most = __uint_as_float(bits);
  const bool zero = most < 7.8886090522101181e-31f;
  inv = zero ? 0.f : __fmul_rn(__frcp_rn(most), AW_E4M3_MAX);
  return zero ? 0.f : __fmul_rn(most, 1.f / AW_E4M3_MAX);
}

// A warp holds a block of 256: elements 4 lane + j and 128 + 4 lane + j.
template <typename T, int MOST>
__global__ void __launch_bounds__(AW_THREADS, 4) psgd_adamw8_kernel(const __grid_constant__ AwArgs<MOST> a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  AW_FOR_CHUNKS(a, t, first, f, steps)
  const long long e0 = (long long)(chunk - first) * AW_CHUNK;
  const uint32_t key = aw_mix(a.h.seed ^ aw_mix((uint32_t)steps));
  const bool wide = ((((uintptr_t)t.m | (uintptr_t)t.v) & 3u) | (((uintptr_t)t.p | (uintptr_t)t.g) & (4 * sizeof(T) - 1))) == 0;
  constexpr int PER_WARP = AW_CHUNK / AW_THREADS / 8;
#pragma unroll 1
  for (int b = 0; b < PER_WARP; ++b) {
    const long long at = e0 + (b * (AW_THREADS / 32) + warp) * AW_BLOCK;
    if (at >= t.n) break;
    const int left = (int)min((long long)AW_BLOCK, t.n - at);
    const long long block = at / AW_BLOCK;
    T* p = (T*)t.p + at;
    const T* g = (const T*)t.g + at;
    uint8_t* m8 = (uint8_t*)t.m + at;
    uint8_t* v8 = (uint8_t*)t.v + at;
    const float ms = t.m_scale[block], vs = t.v_scale[block];
    const bool whole = wide && left == AW_BLOCK;
    float pp[8], gg[8], mm[8], rr[8];
    uint32_t mc[2], vc[2];
    if (whole) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int i = q * 128 + lane * 4;
        aw_load4(g + i, gg + 4 * q);
        aw_load4((const T*)p + i, pp + 4 * q);
        mc[q] = __ldcs(reinterpret_cast<const uint32_t*>(m8 + i));
        vc[q] = __ldcs(reinterpret_cast<const uint32_t*>(v8 + i));
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        mc[q] = vc[q] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = q * 128 + lane * 4 + j;
          const bool in = i < left;
          gg[4 * q + j] = in ? aw_get(g + i) : 0.f;
          pp[4 * q + j] = in ? aw_get(p + i) : 0.f;
          mc[q] |= (in ? (uint32_t)m8[i] : 0u) << (8 * j);
          vc[q] |= (in ? (uint32_t)v8[i] : 0u) << (8 * j);
        }
      }
    }
    uint32_t most_m = 0, most_r = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      aw_decode4(mc[q], ms, mm + 4 * q);
      aw_decode4(vc[q], vs, rr + 4 * q);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v = __fmul_rn(rr[j], rr[j]);
      aw_moments(a.h, gg[j], mm[j], v);
      rr[j] = sqrtf(v);
      pp[j] = aw_update(a.h, f, pp[j], mm[j], rr[j]);
      most_m = max(most_m, __float_as_uint(mm[j]) & 0x7FFFFFFFu);
      most_r = max(most_r, __float_as_uint(rr[j]) & 0x7FFFFFFFu);   // (what is no number may have a sign)
    }
    most_m = __reduce_max_sync(0xffffffffu, most_m);
    most_r = __reduce_max_sync(0xffffffffu, most_r);
    float inv_m, inv_r;
    const float new_ms = aw_scale(most_m, inv_m), new_vs = aw_scale(most_r, inv_r);
    const uint32_t block_key = aw_mix(key ^ (t.block0 + (uint32_t)block));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t random = aw_mix(block_key + (uint32_t)((j >> 2) * 128 + lane * 4 + (j & 3)));
      mm[j] = aw_round(mm[j], inv_m, (random << 4 & 0xFFFF0u) | 8u, false);
      rr[j] = aw_round(rr[j], inv_r, (random >> 12 & 0xFFFF0u) | 8u, true);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      mc[q] = aw_encode4(mm + 4 * q);
      vc[q] = aw_encode4(rr + 4 * q);
      const int i = q * 128 + lane * 4;
      if (whole) {
        aw_store4(p + i, pp + 4 * q);
        __stcs(reinterpret_cast<uint32_t*>(m8 + i), mc[q]);
        __stcs(reinterpret_cast<uint32_t*>(v8 + i), vc[q]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (i + j >= left) continue;
          aw_put(p + i + j, pp[4 * q + j]);
          m8[i + j] = (uint8_t)(mc[q] >> (8 * j));
          v8[i + j] = (uint8_t)(vc[q] >> (8 * j));
        }
      }
    }
    __syncwarp();   // every lane has read the old scales
    if (lane == 0) {
      t.m_scale[block] = new_ms;
      t.v_scale[block] = new_vs;
    }
  }
  }
  aw_count(a);
}

template <typename T, int MOST>
int aw_launch(const AwHyper& h, const PsgdAdamTensor* list, int count, int bits, cudaStream_t stream) {
  AwArgs<MOST> a;
  a.h = h;
  for (int done = 0; done < count;) {
    long long chunks = 0;
    int n = 0;
    for (; n < MOST && done + n < count; ++n) {
      const long long more = (list[done + n].n + AW_CHUNK - 1) / AW_CHUNK;
      if (chunks + more > 0x7fffffffll) {
        if (n > 0) break;
        psgd_set_error("psgd_adamw: a tensor of %lld elements is more than a grid holds", list[done].n);
        return -1;
      }
      chunks += more;
      a.t[n] = list[done + n];
      a.t[n].chunk_end = (uint32_t)chunks;
    }
    a.count = n;
    done += n;
    if (chunks == 0) continue;
    const int grid = (int)(chunks < AW_GRID ? chunks : AW_GRID);
    const int code = bits == 32 ? psgd_launch(psgd_adamw_kernel<T, MOST>, grid, AW_THREADS, 0, stream, 0, a)
                                : psgd_launch(psgd_adamw8_kernel<T, MOST>, grid, AW_THREADS, 0, stream, 0, a);
    if (code) return code;
  }
  return 0;
}

template <typename T>
int aw_dispatch(const AwHyper& h, const PsgdAdamTensor* list, int count, int bits, cudaStream_t stream) {
  if (count <= 40) return aw_launch<T, 40>(h, list, count, bits, stream);
  return aw_launch<T, 400>(h, list, count, bits, stream);
}

}  // namespace

PSGD_API int psgd_adamw_item_bytes() { return (int)sizeof(PsgdAdamTensor); }

// `list`: host memory, read before the call returns. dtype (of p and g): 0 float32, 1 bfloat16, 2 float16. `ticket`: an int of the
// device, zero, that no launch which may run at the same time uses. `lr_at`: a float of the device, or null.
PSGD_API int psgd_adamw_step(const void* list, int count, int dtype, int bits, double lr, const float* lr_at, double beta1, double beta2,
                             double log_beta1, double log_beta2, double eps, double decay, unsigned seed, int* ticket, cudaStream_t stream) {
  if (count <= 0) return 0;
  const AwHyper h = {(float)lr, lr_at, (float)beta1, (float)beta2, (float)(1.0 - beta1), (float)(1.0 - beta2), (float)log_beta1, (float)log_beta2,
                     (float)eps, (float)decay, seed, ticket};
  const PsgdAdamTensor* t = (const PsgdAdamTensor*)list;
  if (dtype == 0) return aw_dispatch<float>(h, t, count, bits, stream);
  if (dtype == 1) return aw_dispatch<__nv_bfloat16>(h, t, count, bits, stream);
  return aw_dispatch<__half>(h, t, count, bits, stream);
}
