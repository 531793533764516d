// AdamW over a list of tensors in one launch, moments in 32 bits or in 8.
//
//   m <- b1 m + (1 - b1) g          v <- b2 v + (1 - b2) g^2          t <- t + 1
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in float32 whatever the type of p and g; p is rounded to its type once. A step moves 28 bytes per float32
// parameter (p, m, v in and out, g in), 16.1 with moments in 8 bits, and computes some tens of operations: the
// memory bounds it in 32 bits (355 M float32 parameters 1444 us, 6.9 TB/s; 31.8 M 135 us, as bfloat16 110 us, 6.4 TB/s). In 8 it is the
// rounding: issue is 62 to 75 % busy, the rest waits for loads (1099 us, 5.2 TB/s; bfloat16 parameters take as long). A block takes 4096 elements of one tensor, found by a search in the list that the launch
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
#include "psgd_pairs.cuh"

namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_CHUNK = 4096;     // elements of a block
constexpr int AW_BLOCK = 256;      // elements that share a scale: one warp, eight per lane
constexpr int AW_PER_SM = 4;       // blocks that run at a time, moments in 8 bits
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
__device__ __forceinline__ void aw_load4(const T* p, float2* f);
template <>
__device__ __forceinline__ void aw_load4<float>(const float* p, float2* f) {
  const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
  f[0] = make_float2(v.x, v.y);
  f[1] = make_float2(v.z, v.w);
}
template <>
__device__ __forceinline__ void aw_load4<__nv_bfloat16>(const __nv_bfloat16* p, float2* f) {
  const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
  f[0] = make_float2(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u));
  f[1] = make_float2(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ void aw_load4<__half>(const __half* p, float2* f) {
  const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
  f[0] = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
  f[1] = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
}
__device__ __forceinline__ void aw_store4(float* p, const float2* f) { __stcs(reinterpret_cast<float4*>(p), make_float4(f[0].x, f[0].y, f[1].x, f[1].y)); }
__device__ __forceinline__ void aw_store4(__nv_bfloat16* p, const float2* f) {
  const __nv_bfloat162 a = __float22bfloat162_rn(f[0]), b = __float22bfloat162_rn(f[1]);
  __stcs(reinterpret_cast<uint2*>(p), make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b)));
}
__device__ __forceinline__ void aw_store4(__half* p, const float2* f) {
  const __half2 a = __float22half2_rn(f[0]), b = __float22half2_rn(f[1]);
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
__device__ __forceinline__ void aw_moments(const AwHyper& h, float2 g, float2& m, float2& v) {
  const float2 m0 = mul2(m, make_float2(h.beta1, h.beta1)), m1 = mul2(g, make_float2(h.rest1, h.rest1));
  const float2 v0 = mul2(v, make_float2(h.beta2, h.beta2)), v1 = mul2(mul2(g, g), make_float2(h.rest2, h.rest2));
  m = make_float2(__fadd_rn(m0.x, m1.x), __fadd_rn(m0.y, m1.y));   // (sums of pairs would be fused with the products)
  v = make_float2(__fadd_rn(v0.x, v1.x), __fadd_rn(v0.y, v1.y));
}
__device__ __forceinline__ float aw_reciprocal(float x) {   // (1 ulp; the update is small beside p)
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 aw_update(const AwHyper& h, const AwFactors& f, float2 p, float2 m, float2 root) {
  const float2 below = fma2(root, make_float2(f.inv_root2, f.inv_root2), make_float2(h.eps, h.eps));
  const float2 u = mul2(m, make_float2(aw_reciprocal(below.x), aw_reciprocal(below.y)));
  return fma2(u, make_float2(-f.size, -f.size), mul2(p, make_float2(f.keep, f.keep)));
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

template <typename T, int MOST>
__global__ void __launch_bounds__(AW_THREADS, 4) psgd_adamw_kernel(const __grid_constant__ AwArgs<MOST> a) {
  const int which = aw_find(a, blockIdx.x, 0);
  const PsgdAdamTensor& t = a.t[which];
  const uint32_t first = which ? a.t[which - 1].chunk_end : 0;
  const long long e0 = (long long)(blockIdx.x - first) * AW_CHUNK;
  const int left = (int)min((long long)AW_CHUNK, t.n - e0);
  T* p = (T*)t.p + e0;
  const T* g = (const T*)t.g + e0;
  float* m = (float*)t.m + e0;
  float* v = (float*)t.v + e0;
  const AwFactors f = aw_factors(a.h, *(volatile const float*)t.step + 1.f);
  const bool wide = ((((uintptr_t)m | (uintptr_t)v) & 15u) | (((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1))) == 0;
  if (wide && left == AW_CHUNK) {
    constexpr int U = 2;
#pragma unroll
    for (int half = 0; half < AW_CHUNK / (AW_THREADS * 4 * U); ++half) {
      float2 pp[U][2], gg[U][2], mm[U][2], vv[U][2];
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
        for (int j = 0; j < 2; ++j) {
          aw_moments(a.h, gg[u][j], mm[u][j], vv[u][j]);
          pp[u][j] = aw_update(a.h, f, pp[u][j], mm[u][j], make_float2(sqrtf(vv[u][j].x), sqrtf(vv[u][j].y)));
        }
        aw_store4(m + i, mm[u]);
        aw_store4(v + i, vv[u]);
        aw_store4(p + i, pp[u]);
      }
    }
  } else {   // the end of a tensor, or one that does not begin on a 16-byte boundary
    for (int i = threadIdx.x; i < left; i += AW_THREADS) {
      float2 mm = make_float2(m[i], 0.f), vv = make_float2(v[i], 0.f);
      aw_moments(a.h, make_float2(aw_get(g + i), 0.f), mm, vv);
      const float2 pp = aw_update(a.h, f, make_float2(aw_get(p + i), 0.f), mm, make_float2(sqrtf(vv.x), 1.f));
      m[i] = mm.x;
      v[i] = vv.x;
      aw_put(p + i, pp.x);
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

__device__ __forceinline__ void aw_decode4(uint32_t codes, float scale, float2* f) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * j)), __NV_E4M3);
    f[j] = mul2(__half22float2(*reinterpret_cast<const __half2*>(&h)), make_float2(scale, scale));
  }
}

// The e4m3 values that two of `x * inv` are rounded to by 16 random bits each. 20 bits of a float's mantissa lie below the three that stay: a random
// number of 20 bits (16, the middle of their step) is added and what lies below is cut. Steps below 2^-6 are those right above it, so
// that range is moved there and back. The conversion to e4m3 is exact but for its saturation. (Where the block holds what is
// no number its scale is none either, whatever the codes are.)
__device__ __forceinline__ float2 aw_round(float2 x, float inv, uint32_t random_x, uint32_t random_y, bool least) {
  const float2 y = mul2(make_float2(fabsf(x.x), fabsf(x.y)), make_float2(inv, inv));
  const float2 shift = make_float2(y.x < 0.015625f ? 0.015625f : 0.f, y.y < 0.015625f ? 0.015625f : 0.f);
  float2 t = add2(y, shift);
  t.x = __uint_as_float((__float_as_uint(t.x) + random_x) & 0xFFF00000u);
  t.y = __uint_as_float((__float_as_uint(t.y) + random_y) & 0xFFF00000u);
  t = make_float2(t.x - shift.x, t.y - shift.y);
  if (least) return make_float2(fmaxf(t.x, y.x > 0.f ? 0.001953125f : 0.f), fmaxf(t.y, y.y > 0.f ? 0.001953125f : 0.f));
  return make_float2(copysignf(t.x, x.x), copysignf(t.y, x.y));
}
__device__ __forceinline__ uint32_t aw_encode4(const float2* f) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(f[0], __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(f[1], __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// The largest magnitude; what is no number wins.
__device__ __forceinline__ float aw_larger(float most, float2 x) {
  asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(fabsf(x.x)), "f"(fabsf(x.y)));
  return most;
}
// Scale of a block from the bits of its largest magnitude. Below 2^-100 a block is taken for zeros: its scale and the reciprocal would leave the normal range.
__device__ __forceinline__ float aw_scale(uint32_t bits, float& inv) {
  const float most = __uint_as_float(bits);
  const bool zero = most < 7.8886090522101181e-31f;
  inv = zero ? 0.f : __fmul_rn(__frcp_rn(most), AW_E4M3_MAX);
  return zero ? 0.f : __fmul_rn(most, 1.f / AW_E4M3_MAX);
}

// A warp holds a block of 256: elements 4 lane + j and 128 + 4 lane + j. A block of threads takes every gridDim.x-th chunk of the list: what it needs
// to know of a tensor it finds out once for most of its chunks. (A step of 355 M float32 parameters: 1256 us so, 2087 with a chunk to a
// block; 6.3 M bfloat16 ones 34 and 41. With 32-bit moments, where there is little to compute, it was the other way round, 1660 and 1459.)
template <typename T, int MOST>
__global__ void __launch_bounds__(AW_THREADS, AW_PER_SM) psgd_adamw8_kernel(const __grid_constant__ AwArgs<MOST> a) {
  constexpr int PER_WARP = AW_CHUNK / AW_THREADS / 8, APART = AW_THREADS / 32 * AW_BLOCK;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int which = -1;
  AwFactors f;
  float steps = 0.f;
  uint32_t first = 0, end = 0, key = 0;
  const uint32_t chunks = a.t[a.count - 1].chunk_end;
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    if (chunk >= end) {
      which = aw_find(a, chunk, which + 1);
      first = which ? a.t[which - 1].chunk_end : 0;
      end = a.t[which].chunk_end;
      const float now = *(volatile const float*)a.t[which].step + 1.f;
      if (now != steps) {
        steps = now;
        f = aw_factors(a.h, steps);
        key = aw_mix(a.h.seed ^ aw_mix((uint32_t)steps));
      }
    }
    const PsgdAdamTensor& t = a.t[which];
    const bool wide = ((((uintptr_t)t.m | (uintptr_t)t.v) & 3u) | (((uintptr_t)t.p | (uintptr_t)t.g) & (4 * sizeof(T) - 1))) == 0;
    const long long at = (long long)(chunk - first) * AW_CHUNK + warp * AW_BLOCK;
    T* p = (T*)t.p + at + lane * 4;
    const T* g = (const T*)t.g + at + lane * 4;
    uint8_t* m8 = (uint8_t*)t.m + at + lane * 4;
    uint8_t* v8 = (uint8_t*)t.v + at + lane * 4;
    float* m_scale = t.m_scale + at / AW_BLOCK;
    float* v_scale = t.v_scale + at / AW_BLOCK;
    const uint32_t block0 = t.block0 + (uint32_t)(at / AW_BLOCK);
    const int rest = (int)min((long long)AW_CHUNK, t.n - at);      // elements of the tensor from the warp's first block on
#pragma unroll 1
    for (int b = 0; b < PER_WARP; ++b) {
      const int left = rest - b * APART;
      if (left <= 0) break;
      const float ms = m_scale[b * (APART / AW_BLOCK)], vs = v_scale[b * (APART / AW_BLOCK)];
      const bool whole = wide && left >= AW_BLOCK;
      float2 pp[4], gg[4], mm[4], rr[4];
      uint32_t mc[2], vc[2];
      if (whole) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int i = b * APART + q * 128;
          aw_load4(g + i, gg + 2 * q);
          aw_load4((const T*)p + i, pp + 2 * q);
          mc[q] = __ldcs(reinterpret_cast<const uint32_t*>(m8 + i));
          vc[q] = __ldcs(reinterpret_cast<const uint32_t*>(v8 + i));
        }
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          mc[q] = vc[q] = 0;
          float x[4], y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = b * APART + q * 128 + j;
            const bool in = q * 128 + lane * 4 + j < left;
            x[j] = in ? aw_get(g + i) : 0.f;
            y[j] = in ? aw_get(p + i) : 0.f;
            mc[q] |= (in ? (uint32_t)m8[i] : 0u) << (8 * j);
            vc[q] |= (in ? (uint32_t)v8[i] : 0u) << (8 * j);
          }
          gg[2 * q] = make_float2(x[0], x[1]), gg[2 * q + 1] = make_float2(x[2], x[3]);
          pp[2 * q] = make_float2(y[0], y[1]), pp[2 * q + 1] = make_float2(y[2], y[3]);
        }
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        aw_decode4(mc[q], ms, mm + 2 * q);
        aw_decode4(vc[q], vs, rr + 2 * q);
      }
      float most_m = 0.f, most_r = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 v = mul2(rr[j], rr[j]);
        aw_moments(a.h, gg[j], mm[j], v);
        rr[j] = make_float2(sqrtf(v.x), sqrtf(v.y));
        pp[j] = aw_update(a.h, f, pp[j], mm[j], rr[j]);
        most_m = aw_larger(most_m, mm[j]);
        most_r = aw_larger(most_r, rr[j]);
      }
      // (as integers the bits of magnitudes order as they do, and what is no number comes last)
      const uint32_t bits_m = __reduce_max_sync(0xffffffffu, __float_as_uint(most_m)), bits_r = __reduce_max_sync(0xffffffffu, __float_as_uint(most_r));
      float inv_m, inv_r;
      const float new_ms = aw_scale(bits_m, inv_m), new_vs = aw_scale(bits_r, inv_r);
      const uint32_t block_key = aw_mix(key ^ (block0 + (uint32_t)b * (APART / AW_BLOCK))) + (uint32_t)lane * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = aw_mix(block_key + (uint32_t)((j >> 1) * 128 + (j & 1) * 2)), y = aw_mix(block_key + (uint32_t)((j >> 1) * 128 + (j & 1) * 2 + 1));
        mm[j] = aw_round(mm[j], inv_m, (x << 4 & 0xFFFF0u) | 8u, (y << 4 & 0xFFFF0u) | 8u, false);
        rr[j] = aw_round(rr[j], inv_r, (x >> 12 & 0xFFFF0u) | 8u, (y >> 12 & 0xFFFF0u) | 8u, true);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        mc[q] = aw_encode4(mm + 2 * q);
        vc[q] = aw_encode4(rr + 2 * q);
        const int i = b * APART + q * 128;
        if (whole) {
          aw_store4(p + i, pp + 2 * q);
          __stcs(reinterpret_cast<uint32_t*>(m8 + i), mc[q]);
          __stcs(reinterpret_cast<uint32_t*>(v8 + i), vc[q]);
        } else {
          const float x[4] = {pp[2 * q].x, pp[2 * q].y, pp[2 * q + 1].x, pp[2 * q + 1].y};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (q * 128 + lane * 4 + j >= left) continue;
            aw_put(p + i + j, x[j]);
            m8[i + j] = (uint8_t)(mc[q] >> (8 * j));
            v8[i + j] = (uint8_t)(vc[q] >> (8 * j));
          }
        }
      }
      __syncwarp();   // every lane has read the old scales
      if (lane == 0) {
        m_scale[b * (APART / AW_BLOCK)] = new_ms;
        v_scale[b * (APART / AW_BLOCK)] = new_vs;
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
    if (chunks == 0) chunks = 1;   // (tensors without elements make steps too: the one block counts them)
    const int grid = (int)(chunks < AW_PER_SM * 148 ? chunks : AW_PER_SM * 148);
    const int code = bits == 32 ? psgd_launch(psgd_adamw_kernel<T, MOST>, (int)chunks, AW_THREADS, 0, stream, 0, a)
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
