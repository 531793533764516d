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
// a number of 64 bits behind the point, whose whole turns fall off by themselves. So it is as exact for far positions as for near ones.
//
// A row is a warp's: its lanes find where the row's sequence begins (32 offsets at a time), compute one angle each, hand them round in
// shared memory, and then take 2 W elements of a head each, W on either side of the pairs, so that a pair lies in one thread. Where there are few
// rows, several warps share one. All heads of a row turn by the same angles: a sine and a cosine for heads * d / (R / 2) elements.
// Sums of weight gradients go from threads to warps to blocks to one more launch, always in the same order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
  float* parts;                    // scratch for these: psgd_rotate_parts floats
  const unsigned long long* frequencies;   // host memory: rotated / 2 fractions of a turn per position
  long long x_row, x_head, grad_row[3], grad_head[3];
  int rows, sequences, heads, keys, values, size, rotated, pairs;
  int type, weight_type;           // 0 float32, 1 bfloat16, 2 float16
  int wide;                        // 64-bit positions
  int norm;
  float eps;
  int pad;
} PsgdRotate;                      // 240 bytes

namespace {

constexpr int RT_THREADS = 256, RT_WARPS = RT_THREADS / 32;
constexpr int RT_MOST_SIZE = 256;
constexpr int RT_SMS = 148;
constexpr int RT_FORWARD_BLOCKS = 3, RT_BACKWARD_BLOCKS = 2;   // of an SM at a time
constexpr float RT_DOWN = 0x1p-70f;                            // for heads whose squares leave the range

struct RtArgs {
  PsgdRotate c;
  int lanes;                       // of a head: a power of two
  int span, parts[2];              // heads of a warp's share of a row, shares of a row's queries and keys
  unsigned long long frequency[RT_MOST_SIZE / 2];
};

// W elements of a type that lie side by side, on a multiple of 16 bytes (or of their size, if that is less).
template <typename T, int W>
struct RtVec;
template <int W>
struct RtVec<float, W> {
  float4 v[W / 4];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) v[i] = __ldcs(reinterpret_cast<const float4*>(p) + i);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) f[4 * i] = v[i].x, f[4 * i + 1] = v[i].y, f[4 * i + 2] = v[i].z, f[4 * i + 3] = v[i].w;
  }
  static __device__ __forceinline__ void store(float* p, const float* f) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
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
__device__ __forceinline__ float2 rt_wide(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ float2 rt_wide(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t rt_narrow(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t rt_narrow(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T, int W>
struct RtVec {
  typedef typename RtWords<W / 2>::type Words;
  union {
    Words v;
    uint32_t w[W / 2];
  };
  __device__ __forceinline__ void load(const T* p) { v = __ldcs(reinterpret_cast<const Words*>(p)); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const float2 p = rt_wide(w[i], T());
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ void store(T* p, const float* f) {
    RtVec o;
#pragma unroll
    for (int i = 0; i < W / 2; ++i) o.w[i] = rt_narrow(f[2 * i], f[2 * i + 1], T());
    *reinterpret_cast<Words*>(p) = o.v;
  }
};

__device__ __forceinline__ float rt_weight(const void* p, int type, int i) {
  if (type == 0) return ((const float*)p)[i];
  if (type == 1) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}

// Position of a row; false where it belongs to no sequence. A whole warp asks. How many offsets are not behind the row: 32 of them at a time,
// evenly apart, which leave a 32nd of the list. (Whatever the list holds, indices stay inside it.)
__device__ __forceinline__ bool rt_position(const PsgdRotate& c, int row, int lane, unsigned long long& position) {
  position = 0;
  if (c.offsets == nullptr) {
    if (c.positions != nullptr) position = c.wide ? ((const unsigned long long*)c.positions)[row] : (unsigned long long)(long long)((const int*)c.positions)[row];
    return true;
  }
  int lo = 0, n = c.sequences + 1;
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
  const int mine = lane < n ? c.offsets[lo + lane] : 0x7fffffff;
  lo += __popc(__ballot_sync(0xffffffffu, lane < n && mine <= row));
  if (lo == 0 || lo > c.sequences) return false;
  position = (unsigned long long)(row - max(c.offsets[lo - 1], 0));
  return true;
}

// Cosine and sine of a fraction of a turn (64 bits behind the point): the nearest quarter is taken out first.
__device__ __forceinline__ float2 rt_angle(unsigned long long turns) {
  const uint32_t high = (uint32_t)(turns >> 32);
  const uint32_t quarter = (high + 0x20000000u) >> 30;
  const int rest = (int)(high - (quarter << 30));
  float s, c;
  sincospif(fmaf((float)rest, 0x1p-31f, (float)(uint32_t)turns * 0x1p-63f), &s, &c);
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  return make_float2((quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b);
}

// What does not change in a thread: its place in a head and the angles that its lane computes.
template <int W, bool PAIRS>
struct RtPlace {
  int slot, heads;           // which of the heads that a warp takes at a time
  int lo, hi, pair;          // its 2 W elements, and the first of its angles
  bool in, turned;
  unsigned long long frequency[RT_MOST_SIZE / 64];
  __device__ __forceinline__ RtPlace(const RtArgs& a) {
    const int lane = threadIdx.x & 31, member = lane & (a.lanes - 1), half = a.c.rotated / 2;
    slot = lane / a.lanes;
    heads = 32 / a.lanes;
    pair = member * W;
    in = 2 * pair < a.c.size;
    if (PAIRS) {
      lo = 2 * pair, hi = lo + W;
      turned = lo < a.c.rotated;
    } else if (pair < half) {
      lo = pair, hi = pair + half;
      turned = true;
    } else {
      lo = a.c.rotated + pair - half, hi = lo + (a.c.size - a.c.rotated) / 2;
      turned = false;
    }
    turned = turned && in;
#pragma unroll
    for (int j = 0; j < RT_MOST_SIZE / 64; ++j) frequency[j] = lane + 32 * j < half ? a.frequency[lane + 32 * j] : 0ull;
  }
  // Cosines and sines of a row's angles, by way of the warp's shared memory.
  __device__ __forceinline__ void angles(const RtArgs& a, unsigned long long position, float2* shared, float* cosine, float* sine) const {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < RT_MOST_SIZE / 64; ++j)
      if (lane + 32 * j < a.c.rotated / 2) shared[lane + 32 * j] = rt_angle(position * frequency[j]);
    __syncwarp();
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const float2 t = turned ? shared[pair + e] : make_float2(1.f, 0.f);
      cosine[e] = t.x, sine[e] = t.y;
    }
  }
  static __device__ __forceinline__ constexpr int first(int e) { return PAIRS ? 2 * e : e; }
  static __device__ __forceinline__ constexpr int second(int e) { return PAIRS ? 2 * e + 1 : W + e; }
  __device__ __forceinline__ int element(int i) const { return i < W ? lo + i : hi + i - W; }
};

// Of the lanes of a head.
__device__ __forceinline__ float rt_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A warp's next share: which of queries (0), keys (1) and values (2), of which row, from which head on.
struct RtShare {
  int kind, row, head, end;
  __device__ __forceinline__ bool at(const RtArgs& a, long long u) {
    const long long queries = (long long)a.c.rows * a.parts[0], keys = (long long)a.c.rows * a.parts[1];
    kind = 0;
    if (u >= queries) {
      u -= queries;
      kind = 1;
      if (u >= keys) {
        kind = 2;
        row = (int)(u - keys);
        return true;
      }
    }
    const int parts = a.parts[kind], have = kind ? a.c.keys : a.c.heads;
    row = parts == 1 ? (int)u : (int)(u / parts);
    head = parts == 1 ? 0 : (int)(u - (long long)row * parts) * a.span;
    end = min(head + a.span, have);
    return true;
  }
};

template <typename T, int W, bool PAIRS>
__global__ void __launch_bounds__(RT_THREADS, RT_FORWARD_BLOCKS) psgd_rotate_kernel(const __grid_constant__ RtArgs a) {
  constexpr int U = 2;       // heads of a thread on their way
  __shared__ float2 s_angles[RT_WARPS][RT_MOST_SIZE / 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const RtPlace<W, PAIRS> place(a);
  const long long shares = (long long)a.c.rows * (a.parts[0] + a.parts[1]);
  const int size = a.c.size;
  for (long long u = (long long)blockIdx.x * RT_WARPS + warp; u < shares; u += (long long)gridDim.x * RT_WARPS) {
    RtShare share;
    share.at(a, u);
    const int have = share.kind ? a.c.keys : a.c.heads;
    const T* x = (const T*)a.c.x + (long long)share.row * a.c.x_row + (share.kind ? (long long)a.c.heads * a.c.x_head : 0);
    T* out = (T*)a.c.out[share.kind] + (long long)share.row * have * size;
    RtVec<T, W> raw[U][2];
    const auto load = [&](int head) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int h = head + j * place.heads + place.slot;
        if (place.in && h < share.end) {
          raw[j][0].load(x + h * a.c.x_head + place.lo);
          raw[j][1].load(x + h * a.c.x_head + place.hi);
        } else {
          raw[j][0].clear();
          raw[j][1].clear();
        }
      }
    };
    load(share.head);
    unsigned long long position;
    const bool held = rt_position(a.c, share.row, lane, position);
    float cosine[W], sine[W], w[2 * W];
    place.angles(a, position, s_angles[warp], cosine, sine);
    const void* weight = a.c.weight[share.kind];
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) w[i] = weight != nullptr && place.in ? rt_weight(weight, a.c.weight_type, place.element(i)) : 1.f;
    for (int head = share.head;;) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float f[2 * W], z[2 * W];
        raw[j][0].unpack(f);
        raw[j][1].unpack(f + W);
        float r = 1.f;
        if (a.c.norm) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 2 * W; ++i) s = fmaf(f[i], f[i], s);
          s = rt_sum(s, a.lanes);
          float eps = a.c.eps;
          const bool large = !(s < 0x1p126f);
          if (__any_sync(0xffffffffu, large)) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * W; ++i) {
              if (large) f[i] *= RT_DOWN;
              t = fmaf(f[i], f[i], t);
            }
            t = rt_sum(t, a.lanes);
            if (large) s = t, eps *= RT_DOWN * RT_DOWN;
          }
          r = rsqrtf(s / (float)size + eps);
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const int p = place.first(e), q = place.second(e);
          const float ya = f[p] * w[p] * r, yb = f[q] * w[q] * r;
          z[p] = ya * cosine[e] - yb * sine[e];
          z[q] = yb * cosine[e] + ya * sine[e];
        }
        const int h = head + j * place.heads + place.slot;
        if (place.in && h < share.end) {
          if (!held) {
#pragma unroll
            for (int i = 0; i < 2 * W; ++i) z[i] = 0.f;
          }
          RtVec<T, W>::store(out + (long long)h * size + place.lo, z);
          RtVec<T, W>::store(out + (long long)h * size + place.hi, z + W);
        }
      }
      head += U * place.heads;
      if (head >= share.end) break;
      load(head);
    }
  }
}

template <typename T, int W, bool PAIRS>
__global__ void __launch_bounds__(RT_THREADS, RT_BACKWARD_BLOCKS) psgd_rotate_grad_kernel(const __grid_constant__ RtArgs a) {
  psgd_launch_dependents();
  __shared__ float2 s_angles[RT_WARPS][RT_MOST_SIZE / 2];
  __shared__ float s_sums[2][RT_WARPS][RT_MOST_SIZE];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, size = a.c.size, all = a.c.heads + a.c.keys + a.c.values;
  const RtPlace<W, PAIRS> place(a);
  const bool sums = a.c.parts != nullptr;
  for (int i = lane; sums && i < 2 * size; i += 32) s_sums[i >= size][warp][i >= size ? i - size : i] = 0.f;
  __syncwarp();
  float acc[2 * W];
#pragma unroll
  for (int i = 0; i < 2 * W; ++i) acc[i] = 0.f;
  // what the warp's threads have added up for one kind
  const auto flush = [&](int kind) {
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) {
      for (int o = a.lanes; o < 32; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
      if (place.slot == 0 && place.in) s_sums[kind][warp][place.element(i)] = acc[i];
      acc[i] = 0.f;
    }
  };
  const long long shares = (long long)a.c.rows * (a.parts[0] + a.parts[1] + (a.c.values && a.c.dx ? 1 : 0));
  int kind = 0;
  for (long long u = (long long)blockIdx.x * RT_WARPS + warp; u < shares; u += (long long)gridDim.x * RT_WARPS) {
    RtShare share;
    share.at(a, u);
    if (share.kind != kind) {
      if (sums && kind < 2) flush(kind);
      kind = share.kind;
    }
    const T* g = (const T*)a.c.grad[kind];
    if (g != nullptr) g += (long long)share.row * a.c.grad_row[kind];
    T* dx = (T*)a.c.dx;
    if (dx != nullptr) dx += ((long long)share.row * all + (kind == 0 ? 0 : kind == 1 ? a.c.heads : a.c.heads + a.c.keys)) * size;
    if (kind == 2) {     // values pass by
      constexpr int N = 16 / (int)sizeof(T);
      const int vectors = size / N;
      for (int i = lane; i < a.c.values * vectors; i += 32) {
        const int h = i / vectors, e = (i - h * vectors) * N;
        *reinterpret_cast<uint4*>(dx + (long long)h * size + e) =
            g != nullptr ? __ldcs(reinterpret_cast<const uint4*>(g + h * a.c.grad_head[2] + e)) : make_uint4(0, 0, 0, 0);
      }
      continue;
    }
    const T* x = (const T*)a.c.x + (long long)share.row * a.c.x_row + (kind ? (long long)a.c.heads * a.c.x_head : 0);
    RtVec<T, W> raw[2], rawg[2];
    const auto load = [&](int head) {
      const int h = head + place.slot;
      if (place.in && h < share.end) {
        raw[0].load(x + h * a.c.x_head + place.lo);
        raw[1].load(x + h * a.c.x_head + place.hi);
      } else {
        raw[0].clear(), raw[1].clear();
      }
      if (place.in && h < share.end && g != nullptr) {
        rawg[0].load(g + h * a.c.grad_head[kind] + place.lo);
        rawg[1].load(g + h * a.c.grad_head[kind] + place.hi);
      } else {
        rawg[0].clear(), rawg[1].clear();
      }
    };
    load(share.head);
    unsigned long long position;
    const bool held = rt_position(a.c, share.row, lane, position);
    float cosine[W], sine[W], w[2 * W];
    place.angles(a, position, s_angles[warp], cosine, sine);
    const void* weight = a.c.weight[kind];
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) w[i] = weight != nullptr && place.in ? rt_weight(weight, a.c.weight_type, place.element(i)) : 1.f;
    for (int head = share.head;;) {
      float f[2 * W], z[2 * W], d[2 * W];
      raw[0].unpack(f), raw[1].unpack(f + W);
      rawg[0].unpack(z), rawg[1].unpack(z + W);
      const int h = head + place.slot;
      const bool mine = place.in && h < share.end;
      head += place.heads;
      const bool more = head < share.end;
      if (more) load(head);
#pragma unroll
      for (int e = 0; e < W; ++e) {     // turned back
        const int p = place.first(e), q = place.second(e);
        d[p] = z[p] * cosine[e] + z[q] * sine[e];
        d[q] = z[q] * cosine[e] - z[p] * sine[e];
      }
      float r = 1.f, t = 0.f, down = 1.f;
      if (a.c.norm) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
          s = fmaf(f[i], f[i], s);
          t = fmaf(d[i] * w[i], f[i], t);
        }
        s = rt_sum(s, a.lanes);
        t = rt_sum(t, a.lanes);
        float eps = a.c.eps;
        const bool large = !(s < 0x1p126f);
        if (__any_sync(0xffffffffu, large)) {
          float s1 = 0.f, t1 = 0.f;
#pragma unroll
          for (int i = 0; i < 2 * W; ++i) {
            if (large) f[i] *= RT_DOWN;
            s1 = fmaf(f[i], f[i], s1);
            t1 = fmaf(d[i] * w[i], f[i], t1);
          }
          s1 = rt_sum(s1, a.lanes);
          t1 = rt_sum(t1, a.lanes);
          if (large) s = s1, t = t1, eps *= RT_DOWN * RT_DOWN, down = RT_DOWN;
        }
        r = rsqrtf(s / (float)size + eps);
        t *= r / (float)size;         // mean(dn n)
      }
      if (mine && held) {
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
          const float n = f[i] * r;
          acc[i] = fmaf(d[i], n, acc[i]);
          z[i] = (d[i] * w[i] - n * t) * (r * down);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) z[i] = 0.f;
      }
      if (mine && dx != nullptr) {
        RtVec<T, W>::store(dx + (long long)h * size + place.lo, z);
        RtVec<T, W>::store(dx + (long long)h * size + place.hi, z + W);
      }
      if (!more) break;
    }
  }
  if (!sums) return;
  if (kind < 2) flush(kind);
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * size; i += RT_THREADS) {
    const int k = i >= size, e = k ? i - size : i;
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < RT_WARPS; ++j) v += s_sums[k][j][e];
    a.c.parts[(long long)blockIdx.x * 2 * size + i] = v;
  }
}

// Sums of the blocks' parts: 32 columns to a block, 8 threads to a column.
__global__ void __launch_bounds__(RT_THREADS) psgd_rotate_weights_kernel(const float* parts, int blocks, int size, int type, void* queries, void* keys) {
  psgd_wait_for_predecessor();
  __shared__ float s_part[RT_WARPS][32];
  const int column = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  float v = 0.f;
  if (column < 2 * size)
    for (int b = slice; b < blocks; b += RT_WARPS) v += __ldcg(parts + (long long)b * 2 * size + column);
  s_part[slice][threadIdx.x & 31] = v;
  __syncthreads();
  if (slice != 0 || column >= 2 * size) return;
#pragma unroll
  for (int j = 1; j < RT_WARPS; ++j) v += s_part[j][threadIdx.x];
  void* out = column < size ? queries : keys;
  const int e = column < size ? column : column - size;
  if (out == nullptr) return;
  if (type == 0) ((float*)out)[e] = v;
  else if (type == 1) ((__nv_bfloat16*)out)[e] = __float2bfloat16_rn(v);
  else ((__half*)out)[e] = __float2half_rn(v);
}

// How a call is spread: 8 elements on either side of the pairs where they fit, shares of rows small enough that every SM has warps, where
// there are few rows.
template <int W>
void rt_plan(RtArgs& a, int warps) {
  int lanes = 1;
  while (lanes * 2 * W < a.c.size) lanes *= 2;
  a.lanes = lanes;
  const int least = 32 / lanes, most = a.c.heads > a.c.keys ? a.c.heads : a.c.keys;
  int steps = (most + least - 1) / least;
  const auto shares = [&](int span) { return (long long)a.c.rows * ((a.c.heads + span - 1) / span + (a.c.keys + span - 1) / span); };
  while (steps > 1 && shares(steps * least) < warps) steps = (steps + 1) / 2;
  a.span = steps * least;
  a.parts[0] = (a.c.heads + a.span - 1) / a.span;
  a.parts[1] = (a.c.keys + a.span - 1) / a.span;
}

template <typename T, int W, bool PAIRS>
int rt_forward(RtArgs& a, cudaStream_t stream) {
  rt_plan<W>(a, RT_SMS * RT_FORWARD_BLOCKS * RT_WARPS);
  const long long shares = (long long)a.c.rows * (a.parts[0] + a.parts[1]), blocks = (shares + RT_WARPS - 1) / RT_WARPS;
  return psgd_launch(psgd_rotate_kernel<T, W, PAIRS>, (int)(blocks < RT_SMS * RT_FORWARD_BLOCKS ? blocks : RT_SMS * RT_FORWARD_BLOCKS), RT_THREADS, 0, stream, 0, a);
}
template <typename T, int W, bool PAIRS>
int rt_backward(RtArgs& a, cudaStream_t stream) {
  rt_plan<W>(a, RT_SMS * RT_BACKWARD_BLOCKS * RT_WARPS);
  const long long shares = (long long)a.c.rows * (a.parts[0] + a.parts[1] + (a.c.values && a.c.dx ? 1 : 0)), blocks = (shares + RT_WARPS - 1) / RT_WARPS;
  const int grid = (int)(blocks < RT_SMS * RT_BACKWARD_BLOCKS ? blocks : RT_SMS * RT_BACKWARD_BLOCKS);
  if (const int code = psgd_launch(psgd_rotate_grad_kernel<T, W, PAIRS>, grid, RT_THREADS, 0, stream, 0, a)) return code;
  if (a.c.parts == nullptr) return 0;
  return psgd_launch(psgd_rotate_weights_kernel, (2 * a.c.size + 31) / 32, RT_THREADS, 0, stream, 1, (const float*)a.c.parts, grid, a.c.size, a.c.weight_type, a.c.dweight[0],
                     a.c.dweight[1]);
}

template <typename T>
int rt_dispatch(RtArgs& a, bool gradient, cudaStream_t stream) {
  const bool wide = a.c.size % 16 == 0 && a.c.rotated % 16 == 0;
  if (a.c.pairs) {
    if (wide) return gradient ? rt_backward<T, 8, true>(a, stream) : rt_forward<T, 8, true>(a, stream);
    return gradient ? rt_backward<T, 4, true>(a, stream) : rt_forward<T, 4, true>(a, stream);
  }
  if (wide) return gradient ? rt_backward<T, 8, false>(a, stream) : rt_forward<T, 8, false>(a, stream);
  return gradient ? rt_backward<T, 4, false>(a, stream) : rt_forward<T, 4, false>(a, stream);
}

int rt_call(const PsgdRotate* call, bool gradient, cudaStream_t stream) {
  if (call->size < 8 || call->size > RT_MOST_SIZE || call->size % 8 || call->rotated < 0 || call->rotated > call->size || call->rotated % 8) {
    psgd_set_error("psgd_rotate: heads of %d of which %d are turned", call->size, call->rotated);
    return PSGD_BAD_ARGUMENT;
  }
  RtArgs a = {};
  a.c = *call;
  for (int i = 0; i < a.c.rotated / 2; ++i) a.frequency[i] = a.c.frequencies[i];
  a.c.frequencies = nullptr;
  if (a.c.type == 0) return rt_dispatch<float>(a, gradient, stream);
  if (a.c.type == 1) return rt_dispatch<__nv_bfloat16>(a, gradient, stream);
  return rt_dispatch<__half>(a, gradient, stream);
}

}  // namespace

PSGD_API int psgd_rotate_call_bytes() { return (int)sizeof(PsgdRotate); }

// Floats of scratch for the gradients of weights.
PSGD_API long long psgd_rotate_parts(int size) { return (long long)RT_SMS * RT_BACKWARD_BLOCKS * 2 * size; }

// `call`: host memory, read before the call returns. Rows that belong to no sequence give zeros.
PSGD_API int psgd_rotate(const PsgdRotate* call, cudaStream_t stream) { return call->rows == 0 ? 0 : rt_call(call, false, stream); }

// The gradients of x (all of it, values included) and of the weights.
PSGD_API int psgd_rotate_grad(const PsgdRotate* call, cudaStream_t stream) { return call->rows == 0 ? 0 : rt_call(call, true, stream); }
