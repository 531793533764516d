// The norm of a list of gradients, taken together, and the same list scaled where it is too large.
//
//   n = (sum_t sum_i g_ti^2)^(1/2)   or   max |g_ti|          c = max_norm / (n + 1e-6)          g <- c g   where not c >= 1
//
// Squares are added in 64 bits: no gradient of 32 bits or less is so large or so small that its square leaves the range, and the order of
// the sums does not show in a norm of 32 bits. (Squares of float64 gradients do from 1.3e154 on, whose norm is infinite, and vanish below 1e-162.) The product is rounded to the gradient's type once. A norm that is no number makes every
// gradient one too; an infinite one makes zeros of the finite ones.
//
// Two launches: sums of blocks, which a second one adds up again in every block, always in the same order. (Lists of up to a megabyte: one, see below.) The list
// travels in the launches' own arguments, so nothing is uploaded and a recorded graph keeps it. A block takes pieces of 16 KiB that begin on
// 16-byte boundaries, wherever a tensor begins: only what a piece's first and last 16 bytes hold of other tensors is left out.
//
// What bounds it is HBM, two reads and a write of everything: 355 M float32 gradients take 204 us for the norm (7.0 TB/s) and 626 with clipping (6.8), as
// bfloat16 118 and 309; 31.8 M float32 25 and 61, where the second read finds a third of them in L2. Squares of 32 bits instead of 64 would save 6 % of a norm of
// 16-bit gradients, whose conversions to 64 bits are then felt, and nothing of float32 ones.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <utility>

#include "psgd_common.cuh"

// One tensor of a list, as the caller fills it in (ops/grad_norm.py).
typedef struct {
  void* g;
  long long n;
  uint32_t type;        // 0 float32, 1 bfloat16, 2 float16, 3 float64
  uint32_t piece_end;   // pieces of the list up to and with this tensor (filled in by the launch)
} PsgdNormTensor;
static_assert(sizeof(PsgdNormTensor) == 24, "as ops/grad_norm.py and host/operators.cpp have it");

namespace {

namespace cg = cooperative_groups;

constexpr int GN_THREADS = 256;
constexpr int GN_PIECE = 16384;                     // bytes
constexpr int GN_VECTORS = GN_PIECE / 16 / GN_THREADS;
constexpr int GN_PER_SM = 6;                        // blocks that run at a time
constexpr int GN_BLOCKS = 148 * GN_PER_SM;          // of a launch, at most
constexpr int GN_PER_SM_LARGE = 4;                  // for more pieces than GN_LARGE, half a gigabyte (355 M float32: 626 us, 631 with six)
constexpr long long GN_LARGE = 32768;
constexpr int GN_CLUSTER = 16, GN_HELD = 4;         // blocks of a short list's one launch, pieces that each holds
constexpr int GN_SMALL_THREADS = GN_PIECE / 16;
constexpr int GN_SHORT = 40, GN_MIDDLE = 320, GN_LONG = 1200;   // tensors of a launch (28.8 KB of arguments; shorter ones are launched sooner)

template <int MOST>
struct GnList {
  int count;
  PsgdNormTensor t[MOST];
};

enum { GN_SQUARES, GN_LARGEST };

// What is joined. As integers the bits of magnitudes are ordered as they are, and what is no number comes last.
template <int KIND>
struct GnPart {
  typedef double type;
  static __device__ __forceinline__ double join(double a, double b) { return a + b; }
  static __device__ __forceinline__ double norm(double a) { return sqrt(a); }
};
template <>
struct GnPart<GN_LARGEST> {
  typedef unsigned long long type;
  static __device__ __forceinline__ type join(type a, type b) { return max(a, b); }
  static __device__ __forceinline__ double norm(type a) { return __longlong_as_double((long long)a); }
};

// What a thread has seen so far.
template <int KIND>
struct GnSeen {
  double sum = 0.0;
  __device__ __forceinline__ void take(float x) { sum = fma((double)x, (double)x, sum); }
  __device__ __forceinline__ void take(double x) { sum = fma(x, x, sum); }
  __device__ __forceinline__ double all() const { return sum; }
};
template <>
struct GnSeen<GN_LARGEST> {
  uint32_t narrow = 0;              // of float32
  unsigned long long wide = 0;
  __device__ __forceinline__ void take(float x) { narrow = max(narrow, __float_as_uint(x) & 0x7fffffffu); }
  __device__ __forceinline__ void take(double x) { wide = max(wide, (unsigned long long)__double_as_longlong(x) & 0x7fffffffffffffffull); }
  __device__ __forceinline__ unsigned long long all() const { return max(wide, (unsigned long long)__double_as_longlong((double)__uint_as_float(narrow))); }
};

template <typename T>
struct GnType;
template <>
struct GnType<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <>
struct GnType<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};
template <>
struct GnType<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float get(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
};
template <>
struct GnType<double> {
  static constexpr int N = 2;
  static __device__ __forceinline__ void unpack(const uint4& r, double* f) {
    f[0] = __hiloint2double((int)r.y, (int)r.x), f[1] = __hiloint2double((int)r.w, (int)r.z);
  }
  static __device__ __forceinline__ uint4 pack(const double* f) {
    return make_uint4((uint32_t)__double2loint(f[0]), (uint32_t)__double2hiint(f[0]), (uint32_t)__double2loint(f[1]), (uint32_t)__double2hiint(f[1]));
  }
  static __device__ __forceinline__ double get(const double* p) { return *p; }
  static __device__ __forceinline__ void put(double* p, double v) { *p = v; }
};
template <typename T>
struct GnWide {
  typedef float type;
};
template <>
struct GnWide<double> {
  typedef double type;
};

// What gradients are multiplied with. One below the normal numbers of 32 bits, for gradients near the end of their range, has few digits left there: two factors then, of
// which the second is at most one, so that nothing vanishes on the way that does not vanish in the end.
struct GnFactor {
  double whole;
  float first, second;
  __device__ __forceinline__ explicit GnFactor(double factor) : whole(factor), first(1.f), second((float)factor) {
    if (factor < 0x1p-126) first = 0x1p-126f, second = (float)(factor * 0x1p126);
  }
  __device__ __forceinline__ float times(float g) const { return g * first * second; }
  __device__ __forceinline__ double times(double g) const { return g * whole; }
};

// Piece `piece` of a tensor: its vectors of 16 bytes lie on 16-byte boundaries, the first one from `base` on; elements [lo, hi) of
// the piece belong to the tensor.
template <typename T>
struct GnPiece {
  T* base;
  int lo, hi;
  __device__ __forceinline__ GnPiece(const PsgdNormTensor& t, uint32_t piece) {
    constexpr int E = GN_PIECE / (int)sizeof(T);
    const int lead = (int)((uintptr_t)t.g & 15u) / (int)sizeof(T);
    const long long first = (long long)piece * E - lead;   // element of the tensor at the piece's beginning
    base = (T*)t.g + first;
    lo = first < 0 ? lead : 0;
    hi = (int)min((long long)E, t.n - first);
  }
};

template <typename T, int KIND>
__device__ __forceinline__ void gn_read(const PsgdNormTensor& t, uint32_t piece, GnSeen<KIND>& seen) {
  typedef GnType<T> V;
  constexpr int N = V::N, E = GN_PIECE / (int)sizeof(T);
  const GnPiece<T> p(t, piece);
  if (p.lo == 0 && p.hi == E) {
    uint4 raw[GN_VECTORS];
#pragma unroll
    for (int i = 0; i < GN_VECTORS; ++i) raw[i] = *reinterpret_cast<const uint4*>(p.base + (i * GN_THREADS + threadIdx.x) * N);
#pragma unroll
    for (int i = 0; i < GN_VECTORS; ++i) {
      typename GnWide<T>::type f[N];
      V::unpack(raw[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) seen.take(f[j]);
    }
    return;
  }
  for (int i = threadIdx.x * N; i < p.hi; i += GN_THREADS * N) {
    if (i >= p.lo && i + N <= p.hi) {
      typename GnWide<T>::type f[N];
      V::unpack(*reinterpret_cast<const uint4*>(p.base + i), f);
#pragma unroll
      for (int j = 0; j < N; ++j) seen.take(f[j]);
    } else {
      for (int j = max(i, p.lo); j < min(i + N, p.hi); ++j) seen.take(V::get(p.base + j));
    }
  }
}

template <typename T>
__device__ __forceinline__ void gn_scale(const PsgdNormTensor& t, uint32_t piece, const GnFactor& c) {
  typedef GnType<T> V;
  typedef typename GnWide<T>::type F;
  constexpr int N = V::N, E = GN_PIECE / (int)sizeof(T);
  const GnPiece<T> p(t, piece);
  if (p.lo == 0 && p.hi == E) {
    uint4 raw[GN_VECTORS];
#pragma unroll
    for (int i = 0; i < GN_VECTORS; ++i) raw[i] = __ldcs(reinterpret_cast<const uint4*>(p.base + (i * GN_THREADS + threadIdx.x) * N));
#pragma unroll
    for (int i = 0; i < GN_VECTORS; ++i) {
      F f[N];
      V::unpack(raw[i], f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = c.times(f[j]);
      __stcs(reinterpret_cast<uint4*>(p.base + (i * GN_THREADS + threadIdx.x) * N), V::pack(f));
    }
    return;
  }
  for (int i = threadIdx.x * N; i < p.hi; i += GN_THREADS * N) {
    if (i >= p.lo && i + N <= p.hi) {
      F f[N];
      V::unpack(*reinterpret_cast<const uint4*>(p.base + i), f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = c.times(f[j]);
      *reinterpret_cast<uint4*>(p.base + i) = V::pack(f);
    } else {
      for (int j = max(i, p.lo); j < min(i + N, p.hi); ++j) V::put(p.base + j, c.times(V::get(p.base + j)));
    }
  }
}

// Of all threads of the block, in thread 0.
template <int KIND>
__device__ __forceinline__ typename GnPart<KIND>::type gn_block(typename GnPart<KIND>::type v) {
  __shared__ typename GnPart<KIND>::type s_part[GN_THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = GnPart<KIND>::join(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < GN_THREADS / 32; ++w) v = GnPart<KIND>::join(v, s_part[w]);
  }
  return v;
}

// The tensor that holds piece `c` of the list, the lo-th or a later one.
template <int MOST>
__device__ __forceinline__ int gn_find(const GnList<MOST>& a, uint32_t c, int lo) {
  int hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c < a.t[mid].piece_end) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

template <int KIND, int MOST>
__global__ void __launch_bounds__(GN_THREADS, GN_PER_SM)
    psgd_grad_norm_kernel(const __grid_constant__ GnList<MOST> a, typename GnPart<KIND>::type* parts, int* taken, int launches) {
  psgd_launch_dependents();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < launches; i += GN_THREADS) taken[i] = 0;
  GnSeen<KIND> seen;
  int which = -1;
  uint32_t first = 0, end = 0;
  const uint32_t pieces = a.t[a.count - 1].piece_end;
  for (uint32_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    if (piece >= end) {
      which = gn_find(a, piece, which + 1);
      first = which ? a.t[which - 1].piece_end : 0;
      end = a.t[which].piece_end;
    }
    const PsgdNormTensor& t = a.t[which];
    if (t.type == 0) gn_read<float, KIND>(t, piece - first, seen);
    else if (t.type == 1) gn_read<__nv_bfloat16, KIND>(t, piece - first, seen);
    else if (t.type == 2) gn_read<__half, KIND>(t, piece - first, seen);
    else gn_read<double, KIND>(t, piece - first, seen);
  }
  const auto acc = gn_block<KIND>(seen.all());
  if (threadIdx.x == 0) parts[blockIdx.x] = acc;
}

// The norm of `count` parts, the same in every block that asks.
template <int KIND>
__device__ __forceinline__ double gn_total(const typename GnPart<KIND>::type* parts, int count) {
  __shared__ double s_norm;
  typename GnPart<KIND>::type v = 0;
  for (int i = threadIdx.x; i < count; i += GN_THREADS) v = GnPart<KIND>::join(v, __ldcg(parts + i));
  v = gn_block<KIND>(v);
  if (threadIdx.x == 0) s_norm = GnPart<KIND>::norm(v);
  __syncthreads();
  return s_norm;
}

__device__ __forceinline__ void gn_write(void* out, int wide, double norm) {
  if (wide) *(double*)out = norm;
  else *(float*)out = (float)norm;
}

template <int KIND>
__global__ void __launch_bounds__(GN_THREADS) psgd_grad_norm_total_kernel(const typename GnPart<KIND>::type* parts, int count, void* out, int wide) {
  psgd_wait_for_predecessor();
  const double norm = gn_total<KIND>(parts, count);
  if (threadIdx.x == 0) gn_write(out, wide, norm);
}

// Pieces are taken in the reverse order, as what was read last may still be in L2, by whichever block is ready: then those under way lie side by side. (355 M
// float32 430 us, 500 with every 888th piece to a block, 530 with a stretch to each. Blocks for one piece each take 6 % less where they scale and
// 100 us where there is nothing to scale.)
template <int KIND, int MOST>
__global__ void __launch_bounds__(GN_THREADS, GN_PER_SM)
    psgd_grad_clip_kernel(const __grid_constant__ GnList<MOST> a, const typename GnPart<KIND>::type* parts, int count, double max_norm, int* taken, void* out, int wide) {
  psgd_launch_dependents();
  psgd_wait_for_predecessor();
  const double norm = gn_total<KIND>(parts, count);
  if (blockIdx.x == 0 && threadIdx.x == 0 && out != nullptr) gn_write(out, wide, norm);
  const double factor = max_norm / (norm + 1e-6);
  if (factor >= 1.0) return;
  const GnFactor c(factor);
  __shared__ uint32_t s_next;
  const uint32_t pieces = a.t[a.count - 1].piece_end;
  const bool more = pieces > gridDim.x;
  int which = 0;
  uint32_t first = 1, end = 0;
  for (uint32_t back = blockIdx.x; back < pieces;) {
    const uint32_t piece = pieces - 1 - back;
    if (more) __syncthreads();
    if (more && threadIdx.x == 0) s_next = gridDim.x + (uint32_t)atomicAdd(taken, 1);
    if (piece < first || piece >= end) {
      which = gn_find(a, piece, 0);
      first = which ? a.t[which - 1].piece_end : 0;
      end = a.t[which].piece_end;
    }
    const PsgdNormTensor& t = a.t[which];
    if (t.type == 0) gn_scale<float>(t, piece - first, c);
    else if (t.type == 1) gn_scale<__nv_bfloat16>(t, piece - first, c);
    else if (t.type == 2) gn_scale<__half>(t, piece - first, c);
    else gn_scale<double>(t, piece - first, c);
    if (!more) return;
    __syncthreads();
    back = s_next;
  }
}

// Short lists in one launch: a cluster of blocks holds all of it in registers, a vector of 16 bytes to a thread and piece. What of a vector
// belongs to other tensors is zero here and is not written back.
template <typename T>
__device__ __forceinline__ uint4 gn_fetch(const GnPiece<T>& p) {
  constexpr int N = GnType<T>::N;
  const int i = threadIdx.x * N;
  if (i >= p.lo && i + N <= p.hi) return *reinterpret_cast<const uint4*>(p.base + i);
  union {
    uint4 v;
    T t[N];
  } raw;
  raw.v = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (i + j >= p.lo && i + j < p.hi) raw.t[j] = p.base[i + j];
  return raw.v;
}
template <typename T, int KIND>
__device__ __forceinline__ void gn_take(const uint4& raw, GnSeen<KIND>& seen) {
  typename GnWide<T>::type f[GnType<T>::N];
  GnType<T>::unpack(raw, f);
#pragma unroll
  for (int j = 0; j < GnType<T>::N; ++j) seen.take(f[j]);
}
template <typename T>
__device__ __forceinline__ void gn_put_back(const GnPiece<T>& p, const uint4& held, const GnFactor& c) {
  typedef typename GnWide<T>::type F;
  constexpr int N = GnType<T>::N;
  const int i = threadIdx.x * N;
  F f[N];
  GnType<T>::unpack(held, f);
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = c.times(f[j]);
  union {
    uint4 v;
    T t[N];
  } raw;
  raw.v = GnType<T>::pack(f);
  if (i >= p.lo && i + N <= p.hi) {
    *reinterpret_cast<uint4*>(p.base + i) = raw.v;
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j >= p.lo && i + j < p.hi) p.base[i + j] = raw.t[j];
  }
}

// (A perceptron's 0.8 MB: 7.2 to 7.5 us to a program that calls it again and again, 9.3 with clusters of 8, 7.8 in two launches. A megabyte: 7.1, 10.3 and 7.7. A few KB: 4.7, 5.3 and
// 7.7. Programs that do more between two calls: 7.6 to 8.2 for the 0.8 MB, by the host.)
template <int KIND, int MOST>
__global__ void __launch_bounds__(GN_SMALL_THREADS, 1)
    psgd_grad_small_kernel(const __grid_constant__ GnList<MOST> a, int clip, double max_norm, void* out, int wide) {
  typedef GnPart<KIND> P;
  __shared__ typename P::type s_warps[GN_SMALL_THREADS / 32], s_parts[GN_CLUSTER];
  __shared__ int s_which[GN_HELD];
  cg::cluster_group cluster = cg::this_cluster();
  auto running = cluster.barrier_arrive();
  const uint32_t pieces = a.t[a.count - 1].piece_end, rank = blockIdx.x;      // (the grid is one cluster)
  if (threadIdx.x < GN_HELD) s_which[threadIdx.x] = rank + threadIdx.x * GN_CLUSTER < pieces ? gn_find(a, rank + threadIdx.x * GN_CLUSTER, 0) : -1;
  __syncthreads();
  uint4 raw[GN_HELD];
#pragma unroll
  for (int i = 0; i < GN_HELD; ++i) {
    const int which = s_which[i];
    raw[i] = make_uint4(0, 0, 0, 0);
    if (which < 0) continue;
    const PsgdNormTensor& t = a.t[which];
    const uint32_t at = rank + i * GN_CLUSTER - (which ? a.t[which - 1].piece_end : 0);
    raw[i] = t.type == 0 ? gn_fetch(GnPiece<float>(t, at)) : t.type == 1 ? gn_fetch(GnPiece<__nv_bfloat16>(t, at)) : t.type == 2 ? gn_fetch(GnPiece<__half>(t, at)) : gn_fetch(GnPiece<double>(t, at));
  }
  GnSeen<KIND> seen;
#pragma unroll
  for (int i = 0; i < GN_HELD; ++i) {
    if (s_which[i] < 0) continue;
    const uint32_t type = a.t[s_which[i]].type;
    if (type == 0) gn_take<float>(raw[i], seen);
    else if (type == 1) gn_take<__nv_bfloat16>(raw[i], seen);
    else if (type == 2) gn_take<__half>(raw[i], seen);
    else gn_take<double>(raw[i], seen);
  }
  typename P::type v = seen.all();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = P::join(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s_warps[threadIdx.x >> 5] = v;
  __syncthreads();
  cluster.barrier_wait(std::move(running));        // all blocks run: their shared memory is there
  if (threadIdx.x < 32) {
    v = s_warps[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = P::join(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (threadIdx.x < GN_CLUSTER) cluster.map_shared_rank(s_parts, threadIdx.x)[rank] = v;
  }
  cluster.sync();
  v = s_parts[0];
#pragma unroll
  for (int i = 1; i < GN_CLUSTER; ++i) v = P::join(v, s_parts[i]);
  const double norm = P::norm(v);
  if (rank == 0 && threadIdx.x == 0) gn_write(out, wide, norm);
  const double factor = max_norm / (norm + 1e-6);
  if (!clip || factor >= 1.0) return;
  const GnFactor c(factor);
#pragma unroll
  for (int i = 0; i < GN_HELD; ++i) {
    const int which = s_which[i];
    if (which < 0) continue;
    const PsgdNormTensor& t = a.t[which];
    const uint32_t at = rank + i * GN_CLUSTER - (which ? a.t[which - 1].piece_end : 0);
    if (t.type == 0) gn_put_back(GnPiece<float>(t, at), raw[i], c);
    else if (t.type == 1) gn_put_back(GnPiece<__nv_bfloat16>(t, at), raw[i], c);
    else if (t.type == 2) gn_put_back(GnPiece<__half>(t, at), raw[i], c);
    else gn_put_back(GnPiece<double>(t, at), raw[i], c);
  }
}

inline long long gn_pieces(const PsgdNormTensor& t) {
  if (t.n <= 0) return 0;
  const long long width = t.type == 0 ? 4 : t.type == 3 ? 8 : 2, lead = (long long)((uintptr_t)t.g & 15u);
  return (lead + t.n * width + GN_PIECE - 1) / GN_PIECE;
}

// The next tensors of a list, as many as a launch takes. Those without elements are left out.
template <int MOST>
int gn_fill(GnList<MOST>& a, const PsgdNormTensor* list, int count, int& done, int& grid) {
  long long pieces = 0;
  a.count = 0;
  for (; done < count && a.count < MOST; ++done) {
    const long long more = gn_pieces(list[done]);
    if (more == 0) continue;
    if (pieces + more > 0x7fffffffll) {
      psgd_set_error("psgd_grad_norm: a list of more than 32 TiB");
      return -1;
    }
    pieces += more;
    a.t[a.count] = list[done];
    a.t[a.count++].piece_end = (uint32_t)pieces;
  }
  const int most = pieces > GN_LARGE ? 148 * GN_PER_SM_LARGE : GN_BLOCKS;
  grid = (int)(pieces < most ? pieces : most);
  return 0;
}

// Does the current device run a cluster of a short list's blocks? (16 of them on one group's SMs are more than every device, or every part of one, has.)
template <int KIND, int MOST>
bool gn_runs_cluster() {
  const auto kernel = psgd_grad_small_kernel<KIND, MOST>;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attrs[2];
  psgd_launch_config(cfg, attrs, GN_CLUSTER, GN_SMALL_THREADS, 0, nullptr, 0, GN_CLUSTER);
  int clusters = 0;
  const bool runs = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                    cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0;
  if (!runs) (void)cudaGetLastError();
  return runs;
}
// Asked once per device (one bit each).
template <int MOST>
bool gn_runs_short() {
  static unsigned long long asked = 0, runs = 0;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  const unsigned long long bit = 1ull << (device & 63);
  if (device < 64 && (__atomic_load_n(&asked, __ATOMIC_ACQUIRE) & bit) != 0) return (__atomic_load_n(&runs, __ATOMIC_RELAXED) & bit) != 0;
  const bool both = gn_runs_cluster<GN_SQUARES, MOST>() && gn_runs_cluster<GN_LARGEST, MOST>();
  if (device < 64) {
    if (both) __atomic_fetch_or(&runs, bit, __ATOMIC_RELAXED);
    __atomic_fetch_or(&asked, bit, __ATOMIC_RELEASE);
  }
  return both;
}

template <int KIND, int MOST>
int gn_run(const PsgdNormTensor* list, int count, int clip, double max_norm, typename GnPart<KIND>::type* parts, void* out, int wide, cudaStream_t stream) {
  typedef const typename GnPart<KIND>::type* Parts;
  GnList<MOST> a;
  int grid = 0, have = 0, launches = 0;
  const int most = (count + MOST - 1) / MOST;       // launches
  int* taken = (int*)(parts + (size_t)most * GN_BLOCKS);
  for (int done = 0; done < count;) {
    if (const int code = gn_fill(a, list, count, done, grid)) return code;
    if (grid == 0) continue;
    if (parts == nullptr) {     // (psgd_grad_norm_parts has found that the device runs it)
      if (launches != 0 || done != count || a.t[a.count - 1].piece_end > GN_CLUSTER * GN_HELD) {
        psgd_set_error("psgd_grad_norm: a list of %d tensors without scratch", count);
        return PSGD_BAD_ARGUMENT;
      }
      return psgd_launch_clusters(psgd_grad_small_kernel<KIND, MOST>, GN_CLUSTER, GN_SMALL_THREADS, 0, stream, 0, GN_CLUSTER, a, clip, max_norm, out, wide);
    }
    if (const int code = psgd_launch(psgd_grad_norm_kernel<KIND, MOST>, grid, GN_THREADS, 0, stream, 0, a, parts + have, taken, clip && launches == 0 ? most : 0)) return code;
    have += grid;
    ++launches;
  }
  if (!clip || launches == 0) return psgd_launch(psgd_grad_norm_total_kernel<KIND>, 1, GN_THREADS, 0, stream, launches > 0, (Parts)parts, have, out, wide);
  if (count <= MOST) return psgd_launch(psgd_grad_clip_kernel<KIND, MOST>, grid, GN_THREADS, 0, stream, 1, a, (Parts)parts, have, max_norm, taken, out, wide);
  for (int done = 0; done < count;) {
    if (const int code = gn_fill(a, list, count, done, grid)) return code;
    if (grid == 0) continue;
    if (const int code = psgd_launch(psgd_grad_clip_kernel<KIND, MOST>, grid, GN_THREADS, 0, stream, 1, a, (Parts)parts, have, max_norm, taken++, out, wide)) return code;
    out = nullptr;
  }
  return 0;
}

template <int KIND>
int gn_dispatch(const PsgdNormTensor* list, int count, int clip, double max_norm, void* parts_at, void* out, int wide, cudaStream_t stream) {
  typename GnPart<KIND>::type* parts = (typename GnPart<KIND>::type*)parts_at;
  if (count <= GN_SHORT) return gn_run<KIND, GN_SHORT>(list, count, clip, max_norm, parts, out, wide, stream);
  if (count <= GN_MIDDLE) return gn_run<KIND, GN_MIDDLE>(list, count, clip, max_norm, parts, out, wide, stream);
  return gn_run<KIND, GN_LONG>(list, count, clip, max_norm, parts, out, wide, stream);
}

}  // namespace

// Words of 8 bytes of scratch that a list asks for on the current device: none where one launch holds it. A list that is given scratch takes two launches.
PSGD_API long long psgd_grad_norm_parts(const void* list, int count) {
  const PsgdNormTensor* t = (const PsgdNormTensor*)list;
  long long pieces = 0;
  for (int i = 0; i < count && pieces <= GN_CLUSTER * GN_HELD; ++i) pieces += gn_pieces(t[i]);
  if (pieces == 0) return 0;
  if (pieces <= GN_CLUSTER * GN_HELD && (count <= GN_SHORT ? gn_runs_short<GN_SHORT>() : count <= GN_MIDDLE ? gn_runs_short<GN_MIDDLE>() : gn_runs_short<GN_LONG>())) return 0;
  return (GN_BLOCKS + 1ll) * (count <= GN_LONG ? 1 : (count + GN_LONG - 1) / GN_LONG);
}

// `list`: host memory, read before the call returns. `largest`: the largest magnitude instead of the root of the sum of squares. `clip`: gradients are
// scaled where max_norm / (norm + 1e-6) is not at least one. `parts`: scratch, null where psgd_grad_norm_parts asked for none. `out`: the norm before that, float, or double where `wide`.
PSGD_API int psgd_grad_norm(const void* list, int count, int largest, int clip, double max_norm, void* parts, void* out, int wide, cudaStream_t stream) {
  const PsgdNormTensor* t = (const PsgdNormTensor*)list;
  if (largest) return gn_dispatch<GN_LARGEST>(t, count, clip, max_norm, parts, out, wide, stream);
  return gn_dispatch<GN_SQUARES>(t, count, clip, max_norm, parts, out, wide, stream);
}
