// Queries and keys of a projection, each head normed and turned by its row's position, forward and backward.
//
//   r = (mean x^2 + eps)^(-1/2)      y = x r w      z_a = y_a cos t - y_b sin t,  z_b = y_b cos t + y_a sin t,   t = position * base^(-2 i / R)
//
// for a head x of d elements, the weights w that all heads of its kind share, and the pairs (a, b) = (i, i + R/2) or (2i, 2i + 1), i < R/2; what
// lies behind the first R elements is not turned. Backward, with dy = the gradient of z turned back, n = x r:
//
//   dw = sum over rows and heads of dy n        dx = r (dn - n mean(dn n)),  dn = dy w
//
// Everything is held in 32 bits; results are rounded to their type once. An angle is a fraction of a turn: the position times the frequency in turns,
// a number of 64 bits behind the point, whose whole turns fall off by themselves. What is left of an angle is
// off by |position| 2^-65 turns, which the rounding of its frequency leaves (less than a float32's rounding up to 2^38), and by 2^-32 that are cut off.
//
// Forward, a row is a warp's: its lanes find where the row's sequence begins (32 offsets at a time), compute one angle each, hand them round in
// shared memory, and then take 2 W elements of a head each, W on either side of the pairs, so that a pair lies in one thread. Where there are few
// rows, several warps share one. All heads of a row turn by the same angles: a sine and a cosine for heads * d / (R / 2) elements. Backward, a warp
// has the same heads of every row that it comes to, queries or keys, whose weight's gradient it adds up. The sums go from threads to warps to blocks
// to one more launch, always in the same order. Inputs come by asynchronous copies into a thread's own places in shared memory, some steps ahead.
//
// 8192 rows of 16 + 16 heads of 64, bfloat16: forward 14.1 us (67 MB, 4.8 TB/s); backward, with 16 heads of values, 25.9 us (134 MB, 5.2 TB/s) and 2 for the
// weights. 14336 rows of 32 + 8 heads of 128: forward 49 us (294 MB, 6.0 TB/s). Besides HBM it is the instructions, some 4 to an element and pass, and
// waiting for shuffles and shared memory: issue is 62 and 57 % busy in the first two.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>
#include <cstddef>
#include <type_traits>

#include "psgd_common.cuh"

// A call, as the caller fills it in (ops/rotary.py, host/operators.cpp). Strides are in elements, of rows and heads.
typedef struct {
  const void* x;                   // [rows, heads + keys + values, size]
  const void* grad[3];             // of queries, keys and values; null: zeros
  const void* weight[2];           // of queries and keys; null: ones
  const int* offsets;              // [sequences + 1], or null
  const void* positions;           // [rows], or null
  void* out[2];                    // queries and keys, contiguous
  void* dx;                        // like x, contiguous, or null
  void* dweight[2];                // of the weights' type, or null
  double* parts;                   // scratch for these: psgd_rotate_parts numbers
  const unsigned long long* frequencies;   // host memory: rotated / 2 fractions of a turn per position
  long long x_row, x_head, grad_row[3], grad_head[3];
  int rows, sequences, heads, keys, values, size, rotated, pairs;
  int type, weight_type;           // 0 float32, 1 bfloat16, 2 float16
  int wide;                        // 64-bit positions
  int norm;
  float eps;
  int pad;
} PsgdRotate;
static_assert(sizeof(PsgdRotate) == 240 && offsetof(PsgdRotate, x_row) == 120 && offsetof(PsgdRotate, rows) == 184, "as ops/rotary.py and host/operators.cpp have it");

// A type's kernels, a file to each, which are compiled side by side. The call's numbers have been checked.
int psgd_rotate_float32(const PsgdRotate* call, bool gradient, cudaStream_t stream);
int psgd_rotate_bfloat16(const PsgdRotate* call, bool gradient, cudaStream_t stream);
int psgd_rotate_float16(const PsgdRotate* call, bool gradient, cudaStream_t stream);

namespace {

constexpr int RT_THREADS = 256, RT_WARPS = RT_THREADS / 32;
constexpr int RT_MOST_SIZE = 256, RT_MOST_ANGLES = RT_MOST_SIZE / 2;
constexpr int RT_MOST_HEADS = 4096;      // (so that the fewest warps that can share a row are no more than RT_PART_BLOCKS have)
constexpr int RT_SMS = 148;
constexpr int RT_FORWARD_BLOCKS = 4, RT_BACKWARD_BLOCKS = 2;      // of an SM at a time
constexpr int RT_FORWARD_STAGES = 3;     // steps whose inputs are on their way or read
constexpr int RT_STEPS = 2;              // of a warp, gradients
constexpr int RT_SUMMED = 32;            // rows of a warp whose products, RT_STEPS to a row, a thread adds up in 32 bits
constexpr int RT_PASSING = 2;            // vectors of values of a thread that pass by with them
// Do the squares of a type leave the range of float32?
template <typename T>
constexpr bool RT_RANGE = !std::is_same<T, __half>::value;
constexpr int RT_PART_BLOCKS = RT_SMS * RT_BACKWARD_BLOCKS;    // that add up gradients of weights
constexpr float RT_DOWN = 0x1p-70f;                            // for heads whose squares leave the range

struct RtArgs {
  PsgdRotate c;
  int lanes;                       // of a head
  int parts[2];                    // warps that share a row's queries, and its keys (a gradient); its queries and keys (forward)
  float share;                     // 1 / size
  unsigned long long frequency[RT_MOST_ANGLES];
};

// Two float32 in one register of 64 bits, so that they need not be moved together before each operation.
typedef unsigned long long RtPair;
__device__ __forceinline__ RtPair rt_pair(float a, float b) {
  RtPair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ RtPair rt_both(float x) { return rt_pair(x, x); }
__device__ __forceinline__ float2 rt_floats(RtPair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ RtPair rt_mul(RtPair a, RtPair b) {
  RtPair c;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c) : "l"(a), "l"(b));
  return c;
}
__device__ __forceinline__ RtPair rt_fma(RtPair a, RtPair b, RtPair c) {
  RtPair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// c - a b (scalars subtract for nothing)
__device__ __forceinline__ RtPair rt_less(RtPair a, RtPair b, RtPair c) {
  const float2 x = rt_floats(a), y = rt_floats(b), z = rt_floats(c);
  return rt_pair(fmaf(-x.x, y.x, z.x), fmaf(-x.y, y.y, z.y));
}

// W elements of a type that lie side by side, on a multiple of 16 bytes (or of their size, if that is less), as W / 2 pairs.
template <typename T, int W>
struct RtVec;
template <int W>
struct RtVec<float, W> {
  float4 v[W / 4];
  static constexpr int BYTES = 4 * W;
  __device__ __forceinline__ void get(const char* p) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) v[i] = reinterpret_cast<const float4*>(p)[i];
  }
  __device__ __forceinline__ void unpack(RtPair* f) const {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) f[2 * i] = rt_pair(v[i].x, v[i].y), f[2 * i + 1] = rt_pair(v[i].z, v[i].w);
  }
  static __device__ __forceinline__ void store(float* p, const RtPair* f) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const float2 a = rt_floats(f[2 * i]), b = rt_floats(f[2 * i + 1]);
      reinterpret_cast<float4*>(p)[i] = make_float4(a.x, a.y, b.x, b.y);
    }
  }
};
template <int N>
struct RtWords;
template <>
struct RtWords<2> {
  typedef uint2 type;
};
template <>
struct RtWords<4> {
  typedef uint4 type;
};
__device__ __forceinline__ RtPair rt_wide(uint32_t w, __nv_bfloat16) { return rt_pair(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ RtPair rt_wide(uint32_t w, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return rt_pair(f.x, f.y);
}
__device__ __forceinline__ uint32_t rt_narrow(float2 f, __nv_bfloat16) {
  const __nv_bfloat162 h = __float22bfloat162_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t rt_narrow(float2 f, __half) {
  const __half2 h = __float22half2_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T, int W>
struct RtVec {
  typedef typename RtWords<W / 2>::type Words;
  union {
    Words v;
    uint32_t w[W / 2];
  };
  static constexpr int BYTES = 2 * W;
  __device__ __forceinline__ void get(const char* p) { v = *reinterpret_cast<const Words*>(p); }
  __device__ __forceinline__ void unpack(RtPair* f) const {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) f[i] = rt_wide(w[i], T());
  }
  static __device__ __forceinline__ void store(T* p, const RtPair* f) {
    RtVec o;
#pragma unroll
    for (int i = 0; i < W / 2; ++i) o.w[i] = rt_narrow(rt_floats(f[i]), T());
    *reinterpret_cast<Words*>(p) = o.v;
  }
};

// What is on its way to a thread's own places in shared memory: WORDS bytes each, zeros where `there` is false (nothing is read then).
template <int BYTES>
__device__ __forceinline__ void rt_fetch(void* to, const void* from, bool there) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(there ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(at), "l"(from), "r"(there ? 8 : 0) : "memory");
}
__device__ __forceinline__ void rt_fetched() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LATER>
__device__ __forceinline__ void rt_await() { asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory"); }

__device__ __forceinline__ float rt_weight(const void* p, int type, int i) {
  if (type == 0) return ((const float*)p)[i];
  if (type == 1) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}

// Where the rows' positions come from. A whole warp asks. How many offsets are not behind the row: 32 of them at a time, evenly apart, which leave a 32nd
// of the list. (Whatever the list holds, indices stay inside it.) The last 32, or a short list, are a lane's each.
struct RtPositions {
  int held;       // a short list's
  bool few;
  __device__ __forceinline__ RtPositions(const PsgdRotate& c) {
    const int lane = threadIdx.x & 31;
    few = c.offsets != nullptr && c.sequences < 32;
    held = few && lane <= c.sequences ? c.offsets[lane] : 0x7fffffff;
  }
  // False where the row belongs to no sequence.
  __device__ __forceinline__ bool of(const PsgdRotate& c, int row, unsigned long long& position) const {
    const int lane = threadIdx.x & 31;
    position = 0;
    if (c.offsets == nullptr) {
      if (c.positions != nullptr) position = c.wide ? ((const unsigned long long*)c.positions)[row] : (unsigned long long)(long long)((const int*)c.positions)[row];
      return true;
    }
    int lo = 0, mine = held;
    if (!few) {
      int n = c.sequences + 1;
      while (n > 32) {
        const int step = (n + 31) >> 5;
        const bool in = lane * step < n;
        const int before = __popc(__ballot_sync(0xffffffffu, in && c.offsets[in ? lo + lane * step : lo] <= row));
        if (before == 0) {                      // (the first of these is behind the row, and so are all)
          n = 0;
          break;
        }
        const int next = (before - 1) * step + 1;
        n = min(step, n - (before - 1) * step) - 1;
        lo += next;
      }
      mine = lane < n ? c.offsets[lo + lane] : 0x7fffffff;
    }
    const unsigned before = __ballot_sync(0xffffffffu, mine <= row);
    const int count = lo + __popc(before);
    if (count == 0 || count > c.sequences) return false;
    // (where the last one that is not behind the row was among these, a lane has it)
    const int start = before ? __shfl_sync(0xffffffffu, mine, (__popc(before) - 1) & 31) : c.offsets[count - 1];
    position = (unsigned long long)(row - max(start, 0));
    return true;
  }
};

// Cosine and sine of a fraction of a turn (64 bits behind the point): the nearest quarter is taken out first. What is left, an eighth of a turn
// at most, goes into the first terms of their series: what follows is below 2e-9 and 3e-10.
__device__ __forceinline__ float2 rt_angle(unsigned long long turns) {
  const uint32_t high = (uint32_t)(turns >> 32);
  const uint32_t quarter = (high + 0x20000000u) >> 30;
  const float t = (float)(int)(high - (quarter << 30)) * 1.4629180792671596e-9f, u = t * t;   // 2 pi / 2^32
  const float s = fmaf(t * u, fmaf(u, fmaf(u, fmaf(u, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), t);
  const float c = fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  return make_float2((quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b);
}

// What a block has in shared memory besides sums.
struct __align__(16) RtShared {
  float cosine[RT_WARPS][RT_MOST_ANGLES], sine[RT_WARPS][RT_MOST_ANGLES];   // of the row that a warp has
  float weight[2][RT_MOST_SIZE];
  unsigned long long frequency[RT_MOST_ANGLES];
  // A thread for each element: `begin`, a barrier, what takes angles, `end`, a barrier, what takes weights. (The weights are on their way meanwhile.)
  __device__ __forceinline__ float2 begin(const RtArgs& a) {
    const int i = threadIdx.x, warp = i >> 5;
    float2 own = make_float2(1.f, 1.f);
    if (i < a.c.size) {
      if (a.c.weight[0] != nullptr) own.x = rt_weight(a.c.weight[0], a.c.weight_type, i);
      if (a.c.weight[1] != nullptr) own.y = rt_weight(a.c.weight[1], a.c.weight_type, i);
    }
    if (i < a.c.rotated / 2) frequency[i] = a.frequency[i];
    for (int j = a.c.rotated / 2 + (i & 31); j < a.c.size / 2; j += 32) cosine[warp][j] = 1.f, sine[warp][j] = 0.f;   // pairs that are not turned
    return own;
  }
  __device__ __forceinline__ void end(const RtArgs& a, float2 own) {
    if (threadIdx.x < a.c.size) weight[0][threadIdx.x] = own.x, weight[1][threadIdx.x] = own.y;
  }
};
static_assert(RT_MOST_HEADS / RT_STEPS + 2 <= RT_PART_BLOCKS * RT_WARPS, "a warp for each share of a row");
static_assert(RT_THREADS >= RT_MOST_SIZE, "a thread for each element of a head");

// Eight, four or two floats of shared memory, on a boundary of 16 bytes or of their size.
template <int W>
__device__ __forceinline__ void rt_get(const float* p, RtPair* f) {
  if (W == 2) f[0] = *reinterpret_cast<const RtPair*>(p);
#pragma unroll
  for (int i = 0; i < W / 4; ++i) {
    const ulonglong2 v = reinterpret_cast<const ulonglong2*>(p)[i];
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}

// A thread's place in a head: W elements from `lo` on and W from `hi` on, which hold W pairs; each of the two lies beside its neighbours' in memory. LANES: of a
// head, where that is known here, or 0: size / 2 W of them.
template <int W, bool PAIRS, int LANES>
struct RtPlace {
  int slot, heads;           // which of the heads that a warp takes at a time
  int lo, hi, member;
  bool in, turned;
  RtPair cosine[W / 2], sine[W / 2];
  static __device__ __forceinline__ int lanes(const RtArgs& a) { return LANES ? LANES : a.lanes; }
  __device__ __forceinline__ RtPlace(const RtArgs& a) {
    const int lane = threadIdx.x & 31, half = a.c.rotated / 2;
    slot = lane / lanes(a);
    member = lane - slot * lanes(a);
    heads = 32 / lanes(a);
    in = slot < heads;
    lo = member * W;
    turned = PAIRS || lo < half;
    if (PAIRS) {
      hi = lo + a.c.size / 2;
    } else if (turned) {
      hi = lo + half;
    } else {
      lo += half;
      hi = lo + (a.c.size - a.c.rotated) / 2;
    }
  }
  // Cosines and sines of a row's angles, by way of the warp's shared memory.
  __device__ __forceinline__ void angles(const RtArgs& a, unsigned long long position, RtShared& shared) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncwarp();
    for (int i = lane; i < a.c.rotated / 2; i += 32) {
      const float2 t = rt_angle(position * shared.frequency[i]);
      shared.cosine[warp][i] = t.x, shared.sine[warp][i] = t.y;
    }
    __syncwarp();
    if (PAIRS) {
      rt_get<W / 2>(shared.cosine[warp] + lo / 2, cosine);
      rt_get<W / 2>(shared.cosine[warp] + hi / 2, cosine + W / 4);
      rt_get<W / 2>(shared.sine[warp] + lo / 2, sine);
      rt_get<W / 2>(shared.sine[warp] + hi / 2, sine + W / 4);
    } else if (turned) {
      rt_get<W>(shared.cosine[warp] + lo, cosine);
      rt_get<W>(shared.sine[warp] + lo, sine);
    } else {
#pragma unroll
      for (int e = 0; e < W / 2; ++e) cosine[e] = rt_both(1.f), sine[e] = rt_both(0.f);
    }
  }
  // Sums over the lanes of a head, N of them side by side (one behind another each would wait for the one before).
  template <int N>
  __device__ __forceinline__ void sums(float (&s)[N], int lanes) const {
    if (LANES && (LANES & (LANES - 1)) == 0) {
#pragma unroll
      for (int o = 1; o < LANES; o <<= 1) {
        float t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = __shfl_xor_sync(0xffffffffu, s[i], o);
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += t[i];
      }
      return;
    }
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < (LANES ? LANES : 32); o <<= 1) {      // (what lies `o` on, as long as that is the same head's)
      if (!LANES && o >= lanes) break;
      float t[N];
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = __shfl_sync(0xffffffffu, s[i], (lane + o) & 31);
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] += member + o < lanes ? t[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __shfl_sync(0xffffffffu, s[i], lane - member);
  }
  __device__ __forceinline__ float sum(float s, int lanes) const {
    float one[1] = {s};
    sums(one, lanes);
    return one[0];
  }
  // The 2 W elements turned, or turned back.
  template <bool BACK>
  __device__ __forceinline__ void turn(RtPair* v) const {
    if (PAIRS) {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float2 p = rt_floats(v[e]), cs = rt_floats(cosine[e / 2]), sn = rt_floats(sine[e / 2]);
        const float c = e & 1 ? cs.y : cs.x, s = e & 1 ? sn.y : sn.x, t = BACK ? -s : s;
        v[e] = rt_pair(fmaf(-p.y, t, p.x * c), fmaf(p.x, t, p.y * c));
      }
    } else {
#pragma unroll
      for (int e = 0; e < W / 2; ++e) {
        const RtPair p = v[e], q = v[W / 2 + e], pc = rt_mul(p, cosine[e]), qc = rt_mul(q, cosine[e]);
        v[e] = BACK ? rt_fma(q, sine[e], pc) : rt_less(q, sine[e], pc);
        v[W / 2 + e] = BACK ? rt_less(p, sine[e], qc) : rt_fma(p, sine[e], qc);
      }
    }
  }
};

__device__ __forceinline__ float rt_two(RtPair p) {
  const float2 f = rt_floats(p);
  return f.x + f.y;
}
template <int W>
__device__ __forceinline__ RtPair rt_dot(const RtPair* a, const RtPair* b) {
  RtPair s = rt_mul(a[0], b[0]);
#pragma unroll
  for (int i = 1; i < W; ++i) s = rt_fma(a[i], b[i], s);
  return s;
}

// A warp takes one row, or a share of it, its steps' inputs some steps ahead.
template <typename T, int W, bool PAIRS, int LANES>
__global__ void __launch_bounds__(RT_THREADS, RT_FORWARD_BLOCKS) psgd_rotate_kernel(const __grid_constant__ RtArgs a) {
  typedef RtVec<T, W> Vec;
  constexpr int HALF = RT_THREADS * Vec::BYTES, STAGE = 2 * HALF;     // of the ring
  __shared__ RtShared shared;
  __shared__ __align__(16) char ring[RT_FORWARD_STAGES * STAGE];
  const int warp = threadIdx.x >> 5, lanes = LANES ? LANES : a.lanes, parts = a.parts[0];
  RtPlace<W, PAIRS, LANES> place(a);
  const int size = a.c.size, all = a.c.heads + a.c.keys, step = place.heads;
  const uint32_t u = blockIdx.x * RT_WARPS + warp;
  int row = (int)u, head = place.slot, end = all;
  if (parts > 1) {
    const int steps = (all + step - 1) / step;
    row = (int)(u / (uint32_t)parts);
    const int part = (int)(u - (uint32_t)row * (uint32_t)parts);
    head += steps * part / parts * step;
    end = min(steps * (part + 1) / parts * step, all);
  }
  const bool live = row < a.c.rows;
  const int count = live ? (end - head + place.slot + step - 1) / step : 0, apart = place.hi - place.lo;
  if (!place.in || !live) end = 0;
  const long long x_step = step * a.c.x_head;
  const T* x = (const T*)a.c.x + (long long)row * a.c.x_row + head * a.c.x_head + place.lo;
  char* const mine = ring + threadIdx.x * Vec::BYTES;
  int ahead = head, to = 0, from = 0;
  const auto fetch = [&]() {      // (lanes without a head, or behind the last one, find zeros)
    rt_fetch<Vec::BYTES>(mine + to, x, ahead < end);
    rt_fetch<Vec::BYTES>(mine + to + HALF, x + apart, ahead < end);
    rt_fetched();
    ahead += step;
    x += x_step;
    to = to == (RT_FORWARD_STAGES - 1) * STAGE ? 0 : to + STAGE;
  };
#pragma unroll
  for (int i = 0; i < RT_FORWARD_STAGES - 1; ++i) fetch();
  const float2 own = shared.begin(a);
  __syncthreads();
  unsigned long long position = 0;
  const bool held = live && RtPositions(a.c).of(a.c, row, position);
  if (held && a.c.rotated > 0) place.angles(a, position, shared);
  shared.end(a, own);
  __syncthreads();
  if (!live) {
    rt_await<0>();
    return;
  }
  const long long out_step = step * size, to_keys = ((T*)a.c.out[1] + ((long long)row * a.c.keys - a.c.heads) * size) - ((T*)a.c.out[0] + (long long)row * a.c.heads * size);
  T* out = (T*)a.c.out[0] + ((long long)row * a.c.heads + head) * size + place.lo;     // (as if the keys lay behind the queries)
  if (!held) {
    RtPair zeros[W / 2];
#pragma unroll
    for (int i = 0; i < W / 2; ++i) zeros[i] = 0;
    for (; head < end; head += step, out += out_step) {
      T* o = head < a.c.heads ? out : out + to_keys;
      Vec::store(o, zeros);
      Vec::store(o + apart, zeros);
    }
    rt_await<0>();
    return;
  }
  const float* weight = shared.weight[0] + place.lo;
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    rt_await<RT_FORWARD_STAGES - 2>();
    Vec raw[2];
    raw[0].get(mine + from), raw[1].get(mine + from + HALF);
    from = from == (RT_FORWARD_STAGES - 1) * STAGE ? 0 : from + STAGE;
    RtPair f[W];
    raw[0].unpack(f), raw[1].unpack(f + W / 2);
    fetch();     // to where the step before this one was read
    const bool key = head >= a.c.heads;
    if (a.c.norm) {
      float s = place.sum(rt_two(rt_dot<W>(f, f)), lanes), eps = a.c.eps;
      if (RT_RANGE<T>) {
        const bool large = !(s < 0x1p126f);
        if (__any_sync(0xffffffffu, large)) {
          const RtPair down = rt_both(large ? RT_DOWN : 1.f);
#pragma unroll
          for (int j = 0; j < W; ++j) f[j] = rt_mul(f[j], down);
          const float t = place.sum(rt_two(rt_dot<W>(f, f)), lanes);
          if (large) s = t, eps *= RT_DOWN * RT_DOWN;
        }
      }
      const RtPair r = rt_both(rsqrtf(fmaf(s, a.share, eps)));
      RtPair w[W];
      const float* of = weight + (key ? RT_MOST_SIZE : 0);
      rt_get<W>(of, w);
      rt_get<W>(of + apart, w + W / 2);
#pragma unroll
      for (int j = 0; j < W; ++j) f[j] = rt_mul(rt_mul(f[j], r), w[j]);
    }
    if (a.c.rotated > 0) place.template turn<false>(f);
    if (head < end) {
      T* o = key ? out + to_keys : out;
      Vec::store(o, f);
      Vec::store(o + apart, f + W / 2);
    }
    head += step;
    out += out_step;
  }
  rt_await<0>();
}

// Do warps that take every `stride`th row have sums of more than RT_SUMMED rows?
__host__ __device__ __forceinline__ bool rt_many_rows(int rows, int stride) { return rows > RT_SUMMED * stride; }

// Gradients: a warp has the same heads of every row that it comes to, RT_STEPS times what its lanes take at once, queries or keys, so that it adds up one weight's
// gradient, and a share of the rows' values, which pass by. Each step has its place in shared memory, which, once read, is filled with the same
// step of the warp's next row.
template <typename T, int W, bool PAIRS, int LANES>
__global__ void __launch_bounds__(RT_THREADS, RT_BACKWARD_BLOCKS) psgd_rotate_grad_kernel(const __grid_constant__ RtArgs a) {
  psgd_launch_dependents();
  typedef RtVec<T, W> Vec;
  constexpr int HALF = RT_THREADS * Vec::BYTES, STEP = 4 * HALF, N = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) char ring[];
  __shared__ RtShared shared;
  __shared__ int s_kind[RT_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, size = a.c.size, lanes = LANES ? LANES : a.lanes;
  RtPlace<W, PAIRS, LANES> place(a);
  const int apart = place.hi - place.lo, step = place.heads, parts = a.parts[0] + a.parts[1];
  const int u = blockIdx.x * RT_WARPS + warp, stride = gridDim.x * RT_WARPS / parts, part = u % parts;
  const int kind = part >= a.parts[0], own = kind ? part - a.parts[0] : part, have = kind ? a.c.keys : a.c.heads, steps = (have + step - 1) / step;
  const int begin = steps * own / a.parts[kind], count = steps * (own + 1) / a.parts[kind] - begin, head = begin * step + place.slot;
  int row = u / parts, ahead = row;
  if (row >= stride) row = ahead = a.c.rows;       // (where the warps are no multiple of the parts)
  const long long x_step = step * a.c.x_head, x_stride = stride * a.c.x_row, g_step = step * a.c.grad_head[kind], g_stride = stride * a.c.grad_row[kind];
  const T* x = (const T*)a.c.x + (long long)row * a.c.x_row + (head + (kind ? a.c.heads : 0)) * a.c.x_head + place.lo;
  const bool given = a.c.grad[kind] != nullptr;
  const T* g = given ? (const T*)a.c.grad[kind] + (long long)row * a.c.grad_row[kind] + head * a.c.grad_head[kind] + place.lo : x;
  char* const mine = ring + threadIdx.x * Vec::BYTES;
  // values: 16 bytes at a time, RT_PASSING of them by way of shared memory as well
  const int all = a.c.heads + a.c.keys + a.c.values, vectors = size / N, passing = a.c.dx != nullptr ? a.c.values * vectors : 0;
  char* const values = ring + RT_STEPS * STEP + threadIdx.x * 16;
  double2* const wide = reinterpret_cast<double2*>(ring + RT_STEPS * STEP + RT_PASSING * RT_THREADS * 16) + threadIdx.x;      // a thread's sums
  const bool valued = a.c.grad[2] != nullptr;
  const T* gv = valued ? (const T*)a.c.grad[2] + (long long)row * a.c.grad_row[2] : x;
  long long passed[RT_PASSING];
#pragma unroll
  for (int j = 0; j < RT_PASSING; ++j) {
    const int i = (j * parts + part) * 32 + lane, h = i / vectors;
    passed[j] = h * a.c.grad_head[2] + (i - h * vectors) * N;
  }
  const long long gv_stride = valued ? stride * a.c.grad_row[2] : 0;
  const auto fetch = [&](int i) {      // (lanes without a head find zeros)
    if (i == 0 && ahead < a.c.rows) {
#pragma unroll
      for (int j = 0; j < RT_PASSING; ++j)
        if ((j * parts + part) * 32 + lane < passing) rt_fetch<16>(values + j * RT_THREADS * 16, gv + passed[j], valued);
    }
    if (i < count && ahead < a.c.rows) {
      const bool there = place.in && head + i * step < have;
      rt_fetch<Vec::BYTES>(mine + i * STEP, x + i * x_step, there);
      rt_fetch<Vec::BYTES>(mine + i * STEP + HALF, x + i * x_step + apart, there);
      rt_fetch<Vec::BYTES>(mine + i * STEP + 2 * HALF, g + i * g_step, there && given);
      rt_fetch<Vec::BYTES>(mine + i * STEP + 3 * HALF, g + i * g_step + apart, there && given);
    }
    rt_fetched();
  };
#pragma unroll
  for (int i = 0; i < RT_STEPS; ++i) fetch(i);
  const bool sums = a.c.parts != nullptr;
  shared.end(a, shared.begin(a));
  __syncthreads();
  const RtPositions positions(a.c);
  T* dx = (T*)a.c.dx + ((long long)row * all + (kind ? a.c.heads : 0) + head) * size + place.lo;
  const long long dx_stride = (long long)stride * all * size;
  const float* weight = shared.weight[kind] + place.lo;
  RtPair acc[W];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = 0;
  if (sums && rt_many_rows(a.c.rows, stride)) {     // (there is room for these sums only then)
#pragma unroll
    for (int i = 0; i < W; ++i) wide[i * RT_THREADS] = make_double2(0.0, 0.0);
  }
  // A thread's sum of the products of RT_SUMMED rows at most is one of 32 bits, of any more of 64 (with 32 all the way a weight's gradient was 2e-7 off for 8192 rows,
  // now 1e-7, and up to 5e-6 for 4 M of them; the sums of 64 wait in shared memory).
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int left = RT_SUMMED; left > 0 && row < a.c.rows; --left, row = ahead) {
      ahead = stride < a.c.rows - row ? row + stride : a.c.rows;
      x += x_stride;
      g += g_stride;
      gv += gv_stride;
      unsigned long long position;
      const bool held = positions.of(a.c, row, position);
      if (a.c.rotated > 0) place.angles(a, position, shared);
#pragma unroll
      for (int i = 0; i < RT_STEPS; ++i) {
        rt_await<RT_STEPS - 1>();
        if (i == 0 && passing > 0) {     // values pass by
          T* o = (T*)a.c.dx + ((long long)row * all + a.c.heads + a.c.keys) * size;
#pragma unroll
          for (int j = 0; j < RT_PASSING; ++j) {
            const int e = (j * parts + part) * 32 + lane;
            if (e < passing) *reinterpret_cast<uint4*>(o + e * N) = *reinterpret_cast<const uint4*>(values + j * RT_THREADS * 16);
          }
          for (int e = (RT_PASSING * parts + part) * 32 + lane; e < passing; e += 32 * parts) {
            const int h = e / vectors;
            *reinterpret_cast<uint4*>(o + e * N) =
                valued ? __ldcs(reinterpret_cast<const uint4*>(gv - gv_stride + h * a.c.grad_head[2] + (e - h * vectors) * N)) : make_uint4(0, 0, 0, 0);
          }
        }
        if (i < count) {
          RtPair f[W], d[W];
          {
            Vec raw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) raw[j].get(mine + i * STEP + j * HALF);
            raw[0].unpack(f), raw[1].unpack(f + W / 2);
            raw[2].unpack(d), raw[3].unpack(d + W / 2);
          }
          fetch(i);
          if (held) {
            if (a.c.rotated > 0) place.template turn<true>(d);
            if (a.c.norm) {
              RtPair w[W];
              rt_get<W>(weight, w);
              rt_get<W>(weight + apart, w + W / 2);
              const auto dots = [&](float& s, float& t) {
                RtPair along = rt_mul(rt_mul(d[0], w[0]), f[0]);
#pragma unroll
                for (int j = 1; j < W; ++j) along = rt_fma(rt_mul(d[j], w[j]), f[j], along);
                float two[2] = {rt_two(rt_dot<W>(f, f)), rt_two(along)};
                place.sums(two, lanes);
                s = two[0], t = two[1];
              };
              float s, t, eps = a.c.eps, down = 1.f;
              dots(s, t);
              if (RT_RANGE<T>) {     // (where only products with gradients leave the range, heads are made smaller that are large enough to stay in it themselves)
                const bool far = !(s < 0x1p126f && fabsf(t) < CUDART_INF_F);
                if (__any_sync(0xffffffffu, far)) {
                  const bool large = far && !(s < 0x1p40f);
                  const RtPair less = rt_both(large ? RT_DOWN : 1.f);
#pragma unroll
                  for (int j = 0; j < W; ++j) f[j] = rt_mul(f[j], less);
                  dots(s, t);
                  if (large) eps *= RT_DOWN * RT_DOWN, down = RT_DOWN;
                }
              }
              const float r = rsqrtf(fmaf(s, a.share, eps));
              const RtPair r2 = rt_both(r), rd = rt_both(r * down), along = rt_both(-t * r * a.share);     // - mean(dn n)
#pragma unroll
              for (int j = 0; j < W; ++j) {
                const RtPair n = rt_mul(f[j], r2);
                acc[j] = rt_fma(d[j], n, acc[j]);
                d[j] = rt_mul(rt_fma(n, along, rt_mul(d[j], w[j])), rd);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < W; ++j) d[j] = 0;
          }
          if (place.in && a.c.dx != nullptr && head + i * step < have) {
            T* o = dx + i * step * size;
            Vec::store(o, d);
            Vec::store(o + apart, d + W / 2);
          }
        } else {
          rt_fetched();
        }
      }
      dx += dx_stride;
    }
    if (row >= a.c.rows) break;
    if (!sums) continue;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float2 own = rt_floats(acc[i]);
      const double2 before = wide[i * RT_THREADS];
      wide[i * RT_THREADS] = make_double2(before.x + own.x, before.y + own.y);
      acc[i] = 0;
    }
  }
  rt_await<0>();
  if (!sums) return;
  __syncthreads();       // (the ring, where the warps' sums go, is free)
  double(*const s_sums)[RT_MOST_SIZE] = reinterpret_cast<double(*)[RT_MOST_SIZE]>(ring);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float2 own = rt_floats(acc[i]);
    double2 v = make_double2(own.x, own.y);
    if (rt_many_rows(a.c.rows, stride)) v.x += wide[i * RT_THREADS].x, v.y += wide[i * RT_THREADS].y;
    if (LANES && (LANES & (LANES - 1)) == 0) {
#pragma unroll
      for (int o = LANES; o < 32; o <<= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
      }
    } else {
      const double2 first = v;
      for (int k = 1; k < place.heads; ++k) {
        v.x += __shfl_sync(0xffffffffu, first.x, (lane + k * lanes) & 31);
        v.y += __shfl_sync(0xffffffffu, first.y, (lane + k * lanes) & 31);
      }
    }
    if (place.slot == 0) *reinterpret_cast<double2*>(&s_sums[warp][(i < W / 2 ? place.lo : place.hi - W) + 2 * i]) = v;
  }
  if (lane == 0) s_kind[warp] = kind;
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * size; i += RT_THREADS) {
    const int k = i >= size, e = k ? i - size : i;
    double v = 0.0;
#pragma unroll
    for (int j = 0; j < RT_WARPS; ++j) v += s_kind[j] == k ? s_sums[j][e] : 0.0;
    a.c.parts[(long long)blockIdx.x * 2 * size + i] = v;
  }
}

// Sums of the blocks' parts: 32 columns to a block, 32 threads to a column.
constexpr int RT_SLICES = 32;
__global__ void __launch_bounds__(32 * RT_SLICES) psgd_rotate_weights_kernel(const double* parts, int blocks, int size, int type, void* queries, void* keys) {
  psgd_wait_for_predecessor();
  __shared__ double s_part[RT_SLICES][32];
  const int column = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  double v = 0.0;
  if (column < 2 * size) {
#pragma unroll
    for (int j = 0; j < (RT_PART_BLOCKS + RT_SLICES - 1) / RT_SLICES; ++j) {
      const int b = j * RT_SLICES + slice;
      v += b < blocks ? __ldcg(parts + (long long)b * 2 * size + column) : 0.0;
    }
  }
  s_part[slice][threadIdx.x & 31] = v;
  __syncthreads();
  if (slice != 0 || column >= 2 * size) return;
#pragma unroll
  for (int j = 1; j < RT_SLICES; ++j) v += s_part[j][threadIdx.x];
  void* out = column < size ? queries : keys;
  const int e = column < size ? column : column - size;
  if (out == nullptr) return;
  if (type == 0) ((float*)out)[e] = (float)v;
  else if (type == 1) ((__nv_bfloat16*)out)[e] = __float2bfloat16_rn((float)v);
  else ((__half*)out)[e] = __float2half_rn((float)v);
}

// How many warps share `heads` of a row: as few as `most` steps to a warp allow, and more where there are few rows, as long as these are `warps` at most.
inline int rt_steps(const RtArgs& a, int heads) {
  const int step = 32 / a.lanes;
  return (heads + step - 1) / step;
}
inline int rt_parts(const RtArgs& a, int heads, int most, long long warps) {
  const int steps = rt_steps(a, heads);
  int parts = (steps + most - 1) / most;
  while (parts < steps && (long long)a.c.rows * (parts + 1) <= warps) ++parts;
  return parts;
}

template <typename T, int W, bool PAIRS, int LANES>
int rt_forward(RtArgs& a, cudaStream_t stream) {
  a.parts[0] = rt_parts(a, a.c.heads + a.c.keys, RT_MOST_HEADS, RT_SMS * RT_FORWARD_BLOCKS * RT_WARPS);
  const long long blocks = ((long long)a.c.rows * a.parts[0] + RT_WARPS - 1) / RT_WARPS;
  return psgd_launch(psgd_rotate_kernel<T, W, PAIRS, LANES>, (int)blocks, RT_THREADS, 0, stream, 0, a);
}
template <typename T, int W, bool PAIRS, int LANES>
int rt_backward(RtArgs& a, cudaStream_t stream) {
  // Half of the warps for either kind, and less where the other kind cannot do with half: every share of a row has a warp of the launch.
  constexpr long long warps = RT_PART_BLOCKS * RT_WARPS;
  const auto left = [&](long long others) { return std::min(warps / 2, warps - a.c.rows * others); };
  a.parts[0] = rt_parts(a, a.c.heads, RT_STEPS, left((rt_steps(a, a.c.keys) + RT_STEPS - 1) / RT_STEPS));
  a.parts[1] = a.c.keys > 0 ? rt_parts(a, a.c.keys, RT_STEPS, left(a.parts[0])) : 0;
  if (a.parts[0] + a.parts[1] > warps) {
    psgd_set_error("psgd_rotate_grad: a row of %d heads of %d wants %d warps", a.c.heads + a.c.keys, a.c.size, a.parts[0] + a.parts[1]);
    return PSGD_BAD_ARGUMENT;
  }
  const long long blocks = ((long long)a.c.rows * (a.parts[0] + a.parts[1]) + RT_WARPS - 1) / RT_WARPS;
  const int grid = (int)(blocks < RT_PART_BLOCKS ? blocks : RT_PART_BLOCKS);
  constexpr size_t ring = (size_t)RT_THREADS * (RT_STEPS * 4 * RtVec<T, W>::BYTES + RT_PASSING * 16), wide = (size_t)RT_THREADS * W * sizeof(double2);
  static_assert(RT_STEPS * 4 * RtVec<T, W>::BYTES >= RT_MOST_SIZE / 32 * (int)sizeof(double), "room for the warps' sums");
  static unsigned long long devices = 0;
  if (const int code = psgd_allow_shared((const void*)psgd_rotate_grad_kernel<T, W, PAIRS, LANES>, ring + wide, devices)) return code;
  const size_t shared = ring + (a.c.parts != nullptr && rt_many_rows(a.c.rows, grid * RT_WARPS / (a.parts[0] + a.parts[1])) ? wide : 0);
  if (const int code = psgd_launch(psgd_rotate_grad_kernel<T, W, PAIRS, LANES>, grid, RT_THREADS, shared, stream, 0, a)) return code;
  if (a.c.parts == nullptr) return 0;
  return psgd_launch(psgd_rotate_weights_kernel, (2 * a.c.size + 31) / 32, 32 * RT_SLICES, 0, stream, 1, (const double*)a.c.parts, grid, a.c.size, a.c.weight_type, a.c.dweight[0],
                     a.c.dweight[1]);
}

template <typename T, int W, bool PAIRS, int LANES>
int rt_launch(RtArgs& a, bool gradient, cudaStream_t stream) {
  return gradient ? rt_backward<T, W, PAIRS, LANES>(a, stream) : rt_forward<T, W, PAIRS, LANES>(a, stream);
}
// Lanes are known at compile time where two heads or more share a warp (16 lanes; L counts down to the call's), and asked for elsewhere, which only heads of more than 128 are, four
// elements to a side. (All sizes from 8 to 256, 2048 elements of queries and keys to a row, known in place of asked: 16384 rows of bfloat16 forward 5 to 17 % shorter, heads of 64 24.8 us in place of 29.8,
// backward 14 % shorter to 3 % longer, heads of 64 48.0 in place of 54.2; 8192 of float32 forward 3 to 7 % shorter, backward 8 % shorter to 1 % longer. Of more than 16 lanes float32
// gains 5 to 8 % forward, and backward between 7 % shorter and, with heads of 256, 7 % longer; twice as many kernels would have to be built for it.)
constexpr int RT_KNOWN_LANES = 16;
template <typename T, int W, bool PAIRS, int L = RT_KNOWN_LANES>
int rt_lanes(RtArgs& a, bool gradient, cudaStream_t stream) {
  // (neighbouring pairs of 16 bits have four to a side where the size is no multiple of 16 only)
  if constexpr (sizeof(T) == 4 || W == 8 || !PAIRS || L % 2 == 1) {
    if (a.lanes == L) return rt_launch<T, W, PAIRS, L>(a, gradient, stream);
  }
  if constexpr (L > 1) return rt_lanes<T, W, PAIRS, L - 1>(a, gradient, stream);
  else if constexpr (2 * W * RT_KNOWN_LANES < RT_MOST_SIZE) return rt_launch<T, W, PAIRS, 0>(a, gradient, stream);
  else return PSGD_BAD_ARGUMENT;      // (no size has other lanes)
}
template <typename T, int W>
int rt_width(RtArgs& a, bool gradient, cudaStream_t stream) {
  a.lanes = a.c.size / (2 * W);
  a.share = 1.f / (float)a.c.size;
  return a.c.pairs ? rt_lanes<T, W, true>(a, gradient, stream) : rt_lanes<T, W, false>(a, gradient, stream);
}
template <typename T>
int rt_dispatch(RtArgs& a, bool gradient, cudaStream_t stream) {
  // Eight elements on either side of the pairs where both fit into vectors of 16 bytes, else four (bfloat16 heads of 64, forward and backward, 8192 rows: 14 and 26 us,
  // with four 18 and 40).
  if constexpr (sizeof(T) == 2) {
    if (a.c.size % 16 == 0 && (a.c.pairs || a.c.rotated % 16 == 0)) return rt_width<T, 8>(a, gradient, stream);
  }
  return rt_width<T, 4>(a, gradient, stream);
}

template <typename T>
int rt_call(const PsgdRotate* call, bool gradient, cudaStream_t stream) {
  RtArgs a = {};
  a.c = *call;
  for (int i = 0; i < a.c.rotated / 2; ++i) a.frequency[i] = a.c.frequencies[i];
  a.c.frequencies = nullptr;
  return rt_dispatch<T>(a, gradient, stream);
}

}  // namespace
