// Log probabilities of given tokens, with the entropy of each row and its most likely tokens, and the gradient.
//
//   log p_t = (z_t - m) / T - log s,   m = max_i z_i,   s = sum_i e_i,   e_i = exp(d_i),   d_i = (z_i - m) / T
//   H       = log s - (sum_i e_i d_i) / s
//   dz_i    = (1 / T) [ g (1[i = t] - p_i) - h p_i (log p_i + H) + sum_j g_j (1[i = i_j] - p_i) ]
//
// for the gradients g, h and g_j of log p_t, H and the log probabilities of the listed tokens i_j. Everything is
// held in 32 bits; inputs are read in their own type and the gradient is rounded to it once. Exponents are taken
// of (z - m) k with k = log2(e) / T, the difference first: a row of the type's lowest value is a uniform
// one, and the error grows with the distance from the maximum only.
//
// The forward pass reads a row once: every thread keeps a running maximum, the sum of exponentials below it and
// the sum of e d, and scales the two when the maximum moves. The gradient is computed elementwise from the row's
// two statistics.
//
// What bounds it is HBM: 8192 x 50257 bfloat16 logits take 136 us forward (6.1 TB/s) and 247 us backward (6.7 TB/s, a read and a write),
// 1920 x 33278 float32 ones 42 us (6.1 TB/s). One exponential per element is a third of what the special function units give in that time.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "psgd_common.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int LP_MAX_TOP = 32;        // one place of a list per lane
constexpr int LP_MAX_CLUSTER = 8;
constexpr float LP_FLOOR = -1e4f;     // exponents below this are zeros; as factors of a zero they must stay finite
constexpr float LP_LN2 = 0.693147180559945309f;

struct LpArgs {
  const void* logits;
  long long row_stride;               // elements between rows
  const void* targets;
  int wide_targets;                   // 64-bit indices
  long long ignore_index;
  int vocab;
  float inv_t, k;                     // 1 / T, log2(e) / T
  int top;
  float* log_probs;
  float2* stats;                      // m, log s of each row
  float* entropy;
  float* top_values;
  long long* top_tokens;
};

__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Vectors of 16 bytes.
template <typename T>
struct LpVec;
template <>
struct LpVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float largest(const uint4& r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <>
struct LpVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
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
  static __device__ __forceinline__ float largest(const uint4& r) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};
template <>
struct LpVec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(h[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
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
  static __device__ __forceinline__ float largest(const uint4& r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
};

__device__ __forceinline__ uint4 lp_load(const void* p) {   // read once: not kept in L1
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// Elements of a row before its first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int lp_lead(const T* row, int vocab) {
  const int lead = (int)((16u - ((uint32_t)(uintptr_t)row & 15u)) & 15u) / (int)sizeof(T);
  return lead < vocab ? lead : vocab;
}

// ---- running statistics of a part of a row -----------------------------------------------------
struct LpSum {
  float m, s, a;   // maximum, sum of e, sum of e d (base 2)
};
__device__ __forceinline__ float lp_base(float m) { return m == -INFINITY ? 0.f : m; }   // what is subtracted: -inf - -inf is no number
template <bool ENT>
__device__ __forceinline__ LpSum lp_join(const LpSum& x, const LpSum& y, float k) {
  LpSum r;
  r.m = fmaxf(x.m, y.m);
  const float b = lp_base(r.m);
  const float dx = (x.m - b) * k, dy = (y.m - b) * k;
  const float fx = lp_exp2(dx), fy = lp_exp2(dy);
  r.s = x.s * fx + y.s * fy;
  r.a = ENT ? (x.a + fmaxf(dx, LP_FLOOR) * x.s) * fx + (y.a + fmaxf(dy, LP_FLOOR) * y.s) * fy : 0.f;
  return r;
}

// ---- lists of the largest ----------------------------------------------------------------------
// A key orders by value, then by the lower index: the bits of the number as an unsigned integer in the order of the numbers, and
// the complement of the index.
__device__ __forceinline__ uint32_t lp_order(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);   // (the two zeros are equal)
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t order) {
  return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ unsigned long long lp_key(float v, int index) {
  return ((unsigned long long)lp_order(v) << 32) | (uint32_t)~index;
}

// The 32 largest keys a warp has seen, in descending order over its lanes. What is not above the k-th of any warp of the
// block (`shared`) cannot be among the k of the row.
struct LpList {
  unsigned long long mine, least;
  __device__ __forceinline__ void init() { mine = 0; least = 0; }
  __device__ __forceinline__ void offer(unsigned long long key, bool valid, int k, unsigned long long* shared) {
    const int lane = threadIdx.x & 31;
    unsigned todo = __ballot_sync(0xffffffffu, valid && key > least);
    if (todo == 0) return;
    bool changed = false;
    while (todo) {
      const int src = __ffs(todo) - 1;
      todo &= todo - 1;
      const unsigned long long c = __shfl_sync(0xffffffffu, key, src);
      if (c <= least) continue;
      const int place = __popc(__ballot_sync(0xffffffffu, mine > c));
      const unsigned long long up = __shfl_up_sync(0xffffffffu, mine, 1);
      mine = lane < place ? mine : lane == place ? c : up;
      const unsigned long long own = __shfl_sync(0xffffffffu, mine, k - 1);
      if (own > least) { least = own; changed = true; }
    }
    if (changed && lane == 0) atomicMax(shared, least);
  }
};

// The `top` largest of a part of a row, in descending order to s_best (zeros behind them), once the part has been read. Every thread brings the
// largest value it has seen; of these, or of groups of them, 32 or 64 values are made. The top-th largest of those is a bound that
// at least `top` elements reach, and few others. The elements of the threads that reach it, a few per cent of the row, are looked through again,
// those of one thread by a whole warp, and what reaches the bound is collected. Where more does than there is room for (equal logits,
// a row that is masked but for a few) every warp keeps a list of all it sees instead: with that alone a batch of 1023 x 33281 float16
// logits took 84 us, without alternatives it takes 14.
constexpr int LP_CANDIDATES = 512;
template <typename T, int THREADS>
__device__ __forceinline__ void lp_select(const T* z, int lead, int v0, int v1, int extra, float most, int top, unsigned long long* s_keys,
                                          unsigned long long* s_best) {
  using V = LpVec<T>;
  constexpr int WARPS = THREADS / 32, KEYS = THREADS < 64 ? 32 : 64, GROUP = THREADS / KEYS, AHEAD = 4;
  __shared__ __align__(16) uint32_t s_most[KEYS];
  __shared__ uint32_t s_bound;
  __shared__ int s_count, s_flagged;
  __shared__ short s_threads[THREADS];
  __shared__ unsigned long long s_least;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t mine = lp_order(most);
  uint32_t group = mine;
#pragma unroll
  for (int o = 1; o < GROUP; o *= 2) group = max(group, __shfl_xor_sync(0xffffffffu, group, o));
  if (tid % GROUP == 0) s_most[tid / GROUP] = group;
  if (tid == 0) {
    s_count = s_flagged = 0;
    s_least = 0;
  }
  if (tid < LP_MAX_TOP) s_best[tid] = 0;
  __syncthreads();
  {   // the place of a group among the groups: its threads compare it with a share each
    constexpr int SHARE = KEYS / GROUP < 4 ? 4 : KEYS / GROUP;
    int above = 0, reach = 0;
#pragma unroll
    for (int i = 0; i < SHARE; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(s_most + tid % GROUP * SHARE + i);
      above += (x.x > group) + (x.y > group) + (x.z > group) + (x.w > group);
      reach += (x.x >= group) + (x.y >= group) + (x.z >= group) + (x.w >= group);
    }
#pragma unroll
    for (int o = 1; o < GROUP; o *= 2) {
      above += __shfl_xor_sync(0xffffffffu, above, o);
      reach += __shfl_xor_sync(0xffffffffu, reach, o);
    }
    if (above < top && reach >= top) s_bound = group;   // (equal ones write the same)
  }
  __syncthreads();
  const uint32_t bound = s_bound;
  const uint4* zv = reinterpret_cast<const uint4*>(z + lead);
  auto take = [&](float v, int index) {
    if (lp_order(v) < bound) return;
    const int at = atomicAdd(&s_count, 1);
    if (at < LP_CANDIDATES) s_keys[at] = lp_key(v, index);
  };
  if (mine >= bound) {
    s_threads[atomicAdd(&s_flagged, 1)] = (short)tid;
    if (extra >= 0) take(V::one(z + extra), extra);
  }
  __syncthreads();
  const int flagged = s_flagged;
  const int per_thread = (v1 - v0 + THREADS - 1) / THREADS;      // vectors, at most
  for (int f = warp * AHEAD; f < flagged; f += WARPS * AHEAD) {
    for (int i = lane; i - lane < per_thread; i += 32) {
      uint4 r[AHEAD];
      int at[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        at[u] = f + u < flagged ? v0 + s_threads[f + u] + i * THREADS : v1;
        if (at[u] < v1) r[u] = zv[at[u]];
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (at[u] >= v1 || lp_order(V::largest(r[u])) < bound) continue;
        float x[V::N];
        V::unpack(r[u], x);
#pragma unroll
        for (int e = 0; e < V::N; ++e) take(x[e], lead + at[u] * V::N + e);
      }
    }
  }
  __syncthreads();
  int count = s_count;
  if (count > LP_CANDIDATES) {
    __syncthreads();
    LpList list;
    list.init();
    for (int v = v0 + tid; v - tid < v1; v += THREADS) {
      const bool valid = v < v1;
      uint4 r = make_uint4(0, 0, 0, 0);
      if (valid) r = zv[v];
      // (one lane's reading for all: others raise it meanwhile, and lanes that held different bounds would part in front of votes of the whole warp)
      const unsigned long long seen = __shfl_sync(0xffffffffu, *(volatile unsigned long long*)&s_least, 0);
      if (seen > list.least) list.least = seen;
      if (!__any_sync(0xffffffffu, valid && lp_order(V::largest(r)) >= (uint32_t)(list.least >> 32))) continue;
      float f[V::N];
      V::unpack(r, f);
#pragma unroll
      for (int i = 0; i < V::N; ++i) list.offer(lp_key(f[i], lead + v * V::N + i), valid, top, &s_least);
    }
    list.offer(extra >= 0 ? lp_key(V::one(z + extra), extra) : 0, extra >= 0, top, &s_least);
    s_keys[tid] = lane < top ? list.mine : 0;
    count = THREADS;
    __syncthreads();
  }
  for (int c = tid; c < count; c += THREADS) {   // a key's place is the number of larger ones
    const unsigned long long key = s_keys[c];
    int place = 0;
#pragma unroll 4
    for (int i = 0; i < count; ++i) place += s_keys[i] > key;
    if (key != 0 && place < top) s_best[place] = key;
  }
  __syncthreads();
}

template <typename T, int THREADS, bool TOP, bool ENT>
__global__ void __launch_bounds__(THREADS) psgd_token_logprob_kernel(const __grid_constant__ LpArgs a) {
  using V = LpVec<T>;
  constexpr int U = sizeof(T) == 4 ? 8 : 4, WARPS = THREADS / 32;
  __shared__ LpSum s_sum[WARPS];
  __shared__ LpSum s_parts[LP_MAX_CLUSTER];
  __shared__ unsigned long long s_keys[TOP ? LP_CANDIDATES : 1], s_best[TOP ? LP_MAX_TOP : 1];
  __shared__ unsigned long long s_cluster_keys[TOP ? LP_MAX_CLUSTER * LP_MAX_TOP : 1];

  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* z = (const T*)a.logits + row * a.row_stride;
  const long long target = a.wide_targets ? ((const long long*)a.targets)[row] : (long long)((const int*)a.targets)[row];
  const bool ignored = target == a.ignore_index;
  if (!TOP && !ENT && ignored) {   // nothing of this row is asked for (the same for all CTAs of its cluster)
    if (part == 0 && tid == 0) {
      a.log_probs[row] = 0.f;
      a.stats[row] = make_float2(0.f, 0.f);
    }
    return;
  }
  // Said here and waited for behind the row: all CTAs of the cluster run, so that the shared memory of the first may be written.
  if (parts > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  const bool known = target >= 0 && target < a.vocab;
  float z_target = 0.f;
  if (part == 0 && tid == 0 && known) z_target = V::one(z + target);   // on its way while the row is read
  const int lead = lp_lead(z, a.vocab);
  const int nvec = (a.vocab - lead) / V::N;
  const int share = (nvec + parts - 1) / parts;
  const int v0 = min(part * share, nvec), v1 = min(v0 + share, nvec);
  const uint4* zv = reinterpret_cast<const uint4*>(z + lead);

  LpSum t = {-INFINITY, 0.f, 0.f};
  auto move_to = [&](float m) {   // the maximum moves to m
    if (m > t.m) {
      const float d = (t.m - m) * a.k, f = lp_exp2(d);
      if (ENT) t.a = (t.a + fmaxf(d, LP_FLOOR) * t.s) * f;
      t.s *= f;
      t.m = m;
    }
  };
  auto add = [&](float v, float b) {
    const float d = (v - b) * a.k, e = lp_exp2(d);
    t.s += e;
    if (ENT) t.a = fmaf(e, fmaxf(d, LP_FLOOR), t.a);
  };
  int v = v0 + tid;
  for (; v - tid + U * THREADS <= v1; v += U * THREADS) {
    uint4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = lp_load(zv + v + u * THREADS);
    float most[U];
#pragma unroll
    for (int u = 0; u < U; ++u) most[u] = V::largest(r[u]);
    float largest = most[0];
#pragma unroll
    for (int u = 1; u < U; ++u) largest = fmaxf(largest, most[u]);
    move_to(largest);
    const float b = lp_base(t.m);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[V::N];
      V::unpack(r[u], f);
#pragma unroll
      for (int i = 0; i < V::N; ++i) add(f[i], b);
    }
  }
  for (; v < v1; v += THREADS) {
    const uint4 r = lp_load(zv + v);
    move_to(V::largest(r));
    const float b = lp_base(t.m);
    float f[V::N];
    V::unpack(r, f);
#pragma unroll
    for (int i = 0; i < V::N; ++i) add(f[i], b);
  }
  // what lies before the first and behind the last whole vector: at most 14 elements, in warp 0
  int extra = -1;
  if (warp == 0) {
    const int tail0 = lead + nvec * V::N, tail = a.vocab - tail0;
    if (part == 0 && lane < lead) extra = lane;
    if (part == parts - 1 && lane >= 16 && lane - 16 < tail) extra = tail0 + lane - 16;
    if (extra >= 0) {
      const float f = V::one(z + extra);
      move_to(f);
      add(f, lp_base(t.m));
    }
  }
  if (TOP) lp_select<T, THREADS>(z, lead, v0, v1, extra, t.m, a.top, s_keys, s_best);

  // over the warp, the block, the cluster
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpSum y;
    y.m = __shfl_xor_sync(0xffffffffu, t.m, o);
    y.s = __shfl_xor_sync(0xffffffffu, t.s, o);
    y.a = ENT ? __shfl_xor_sync(0xffffffffu, t.a, o) : 0.f;
    t = lp_join<ENT>(t, y, a.k);
  }
  if (lane == 0) s_sum[warp] = t;
  __syncthreads();
  if (parts > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w) t = lp_join<ENT>(t, s_sum[w], a.k);
    if (parts > 1) *cluster.map_shared_rank(&s_parts[part], 0) = t;
  }
  if (parts > 1) {
    if (TOP && tid < a.top) *cluster.map_shared_rank(&s_cluster_keys[part * LP_MAX_TOP + tid], 0) = s_best[tid];
    cluster.sync();
    if (part != 0) return;
    if (TOP) {
      if (tid < LP_MAX_TOP) s_best[tid] = 0;
      __syncthreads();
      for (int c = tid; c < parts * LP_MAX_TOP; c += THREADS) {
        if ((c & 31) >= a.top) continue;
        const unsigned long long key = s_cluster_keys[c];
        int place = 0;
        for (int w = 0; w < parts; ++w)
          for (int j = 0; j < a.top; ++j) place += s_cluster_keys[w * LP_MAX_TOP + j] > key;
        if (key != 0 && place < a.top) s_best[place] = key;
      }
    }
    if (tid == 0)
      for (int p = 1; p < parts; ++p) t = lp_join<ENT>(t, s_parts[p], a.k);
  }
  // every thread that writes needs m and log s
  if (tid == 0) {
    const bool empty = t.m == -INFINITY && t.s == 0.f;   // every token is masked: there is no distribution
    const float log_s = empty ? 0.f : logf(t.s);
    s_sum[0] = {t.m, log_s, 0.f};
    a.stats[row] = make_float2(t.m, log_s);
    a.log_probs[row] = ignored ? 0.f : !known ? NAN : empty ? -INFINITY : (z_target - t.m) * a.inv_t - log_s;
    if (ENT) a.entropy[row] = empty ? 0.f : log_s - LP_LN2 * (t.a / t.s);
  }
  if (TOP) {
    __syncthreads();
    if (tid < a.top) {
      const unsigned long long key = s_best[tid];
      const float m = s_sum[0].m, log_s = s_sum[0].s;
      const float value = lp_value((uint32_t)(key >> 32));
      // (a row that holds what is not a number has fewer keys than places)
      a.top_tokens[row * a.top + tid] = key == 0 ? 0 : (long long)(int)~(uint32_t)key;
      a.top_values[row * a.top + tid] = key == 0 ? NAN : m == -INFINITY && log_s == 0.f ? -INFINITY : (value - m) * a.inv_t - log_s;
    }
  }
}

// ---- gradient ----------------------------------------------------------------------------------
struct LpGradArgs {
  const void* logits;
  long long row_stride;
  void* grad;                         // rows of grad_stride elements that lie on 16-byte boundaries where those of the logits do
  long long grad_stride;
  const void* targets;
  int wide_targets;
  long long ignore_index;
  long long rows;
  int vocab, chunks;                  // chunks of a row
  float inv_t, k;
  int top;
  const float2* stats;
  const float* entropy;
  const long long* top_tokens;
  const float* g_log_prob;            // each may be null
  const float* g_entropy;
  const float* g_top;
};

constexpr int LG_THREADS = 256, LG_U = 4;

// One chunk of a row per block: elementwise, so nothing waits for anything.
template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(LG_THREADS) psgd_token_logprob_grad_kernel(const __grid_constant__ LpGradArgs a) {
  using V = LpVec<T>;
  const int tid = threadIdx.x;
  const long long row = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x - row * a.chunks);
  const T* z = (const T*)a.logits + row * a.row_stride;
  T* dz = (T*)a.grad + row * a.grad_stride;
  const long long target = a.wide_targets ? ((const long long*)a.targets)[row] : (long long)((const int*)a.targets)[row];
  const bool ignored = target == a.ignore_index;
  const float2 st = a.stats[row];
  const float m = st.x, log_s = st.y;
  const bool empty = m == -INFINITY && log_s == 0.f;
  float g = a.g_log_prob && !ignored ? a.g_log_prob[row] : 0.f;
  if (a.g_log_prob && !ignored && (target < 0 || target >= a.vocab)) g = NAN;   // (entropy and alternatives do not depend on the target)
  float all = g;
  if (TOP)
    for (int j = 0; j < a.top; ++j) all += a.g_top[row * a.top + j];
  const float h = ENT ? a.g_entropy[row] : 0.f;
  const float c1 = ENT ? -(all + h * a.entropy[row]) * a.inv_t : -all * a.inv_t;
  const float c2 = -h * LP_LN2 * a.inv_t;
  const float base = lp_base(m), log2_s = log_s * (1.f / LP_LN2);
  const bool zeros = empty || (!ENT && !TOP && ignored);   // no gradient: the row is not read
  const int at = ignored || target < 0 || target >= a.vocab ? -1 : (int)target;
  const float g_at = g * a.inv_t;
  auto slope = [&](float v) {
    const float x = fmaf(v - base, a.k, -log2_s), p = lp_exp2(x);
    return p * (ENT ? fmaf(c2, fmaxf(x, LP_FLOOR), c1) : c1);
  };
  auto element = [&](int i) {
    float d = zeros ? 0.f : slope(V::one(z + i));
    if (i == at && !empty) d += g_at;
    return d;
  };

  const int lead = lp_lead(z, a.vocab), nvec = (a.vocab - lead) / V::N;
  const int v0 = chunk * (LG_THREADS * LG_U);
  const uint4* zv = reinterpret_cast<const uint4*>(z + lead);
  uint4* dv = reinterpret_cast<uint4*>(dz + lead);
  uint4 r[LG_U];
#pragma unroll
  for (int u = 0; u < LG_U; ++u) {
    const int v = v0 + u * LG_THREADS + tid;
    if (!zeros && v < nvec) r[u] = lp_load(zv + v);
  }
#pragma unroll
  for (int u = 0; u < LG_U; ++u) {
    const int v = v0 + u * LG_THREADS + tid;
    if (v >= nvec) continue;
    float f[V::N];
    if (zeros) {
#pragma unroll
      for (int i = 0; i < V::N; ++i) f[i] = 0.f;
    } else {
      V::unpack(r[u], f);
#pragma unroll
      for (int i = 0; i < V::N; ++i) f[i] = slope(f[i]);
      const int in = at - lead - v * V::N;
      if ((unsigned)in < (unsigned)V::N) {
#pragma unroll
        for (int i = 0; i < V::N; ++i) f[i] += i == in ? g_at : 0.f;
      }
    }
    dv[v] = V::pack(f);
  }
  // what no whole vector covers, by the first block of the row
  const int tail0 = lead + nvec * V::N;
  if (chunk == 0) {
    if (tid < lead) V::put(dz + tid, element(tid));
    const int i = tail0 + tid - 32;
    if (tid >= 32 && i < a.vocab) V::put(dz + i, element(i));
  }
  if (TOP) {
    // The listed tokens once more, each with all that it gets: one rounding, whatever coincides. The block that wrote an element
    // writes it again.
    __syncthreads();
    if (tid < a.top && !zeros) {
      const int i = (int)a.top_tokens[row * a.top + tid];
      const int v = i < lead || i >= tail0 ? 0 : (i - lead) / V::N;
      if (i >= 0 && i < a.vocab && v / (LG_THREADS * LG_U) == chunk) V::put(dz + i, element(i) + a.g_top[row * a.top + tid] * a.inv_t);
    }
  }
}

template <typename T, int THREADS>
int lp_forward(const LpArgs& a, long long rows, int cluster, cudaStream_t stream) {
  const bool top = a.top > 0, ent = a.entropy != nullptr;
  auto kernel = top ? (ent ? psgd_token_logprob_kernel<T, THREADS, true, true> : psgd_token_logprob_kernel<T, THREADS, true, false>)
                    : (ent ? psgd_token_logprob_kernel<T, THREADS, false, true> : psgd_token_logprob_kernel<T, THREADS, false, false>);
  return psgd_launch_clusters(kernel, (int)(rows * cluster), THREADS, 0, stream, 0, cluster, a);
}

template <typename T>
int lp_dispatch(const LpArgs& a, long long rows, cudaStream_t stream) {
  // Short rows: a warp each, without barriers; with many alternatives two, since the bound of 32 values is a low one where most of them are
  // asked for (16384 x 1000 float16: 15 us by one warp, 17 by two; with 8 alternatives 45 and 45, with 20 86 and 52).
  if (a.vocab * (long long)sizeof(T) <= 4096 && a.top <= 8) return lp_forward<T, 32>(a, rows, 1, stream);
  if (a.vocab * (long long)sizeof(T) <= 8192) return lp_forward<T, 64>(a, rows, 1, stream);
  // Few rows: a cluster shares one, so that the row is read by several SMs at a time.
  int cluster = 1;
  while (cluster < LP_MAX_CLUSTER && rows * cluster < 296 && a.vocab / (2 * cluster) >= 2048) cluster *= 2;
  return lp_forward<T, 256>(a, rows, cluster, stream);
}

template <typename T>
int lp_grad_dispatch(LpGradArgs& a, cudaStream_t stream) {
  const int per_block = LG_THREADS * LG_U * LpVec<T>::N;
  a.chunks = (a.vocab + per_block - 1) / per_block;
  if (a.rows * a.chunks > 0x7fffffffll) {
    psgd_set_error("psgd_token_logprob_grad: %lld rows of %d elements are more blocks than a grid holds", a.rows, a.vocab);
    return -1;
  }
  const bool ent = a.g_entropy != nullptr, top = a.g_top != nullptr;
  auto kernel = top ? (ent ? psgd_token_logprob_grad_kernel<T, true, true> : psgd_token_logprob_grad_kernel<T, false, true>)
                    : (ent ? psgd_token_logprob_grad_kernel<T, true, false> : psgd_token_logprob_grad_kernel<T, false, false>);
  return psgd_launch(kernel, (int)(a.rows * a.chunks), LG_THREADS, 0, stream, 0, a);
}

}  // namespace

PSGD_API int psgd_token_logprob_max_top() { return LP_MAX_TOP; }

// dtype: 0 float32, 1 bfloat16, 2 float16. Outputs but log_probs and stats may be null (top_values and top_tokens with top = 0).
PSGD_API int psgd_token_logprob(const void* logits, int dtype, long long rows, int vocab, long long row_stride, const void* targets,
                                int wide_targets, long long ignore_index, float inv_t, int top, float* log_probs, float* stats,
                                float* entropy, float* top_values, long long* top_tokens, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (vocab < 1 || top < 0 || top > LP_MAX_TOP || top > vocab || rows > 0x7fffffffll / LP_MAX_CLUSTER) {
    psgd_set_error("psgd_token_logprob: %lld rows of %d elements, %d largest", rows, vocab, top);
    return -1;
  }
  LpArgs a = {logits, row_stride, targets, wide_targets, ignore_index, vocab, inv_t, inv_t * (1.f / LP_LN2), top, log_probs, (float2*)stats,
              entropy, top_values, top_tokens};
  if (dtype == 0) return lp_dispatch<float>(a, rows, stream);
  if (dtype == 1) return lp_dispatch<__nv_bfloat16>(a, rows, stream);
  return lp_dispatch<__half>(a, rows, stream);
}

// `grad` has rows of grad_stride elements; every row of it lies as far from a 16-byte boundary as that of the logits.
PSGD_API int psgd_token_logprob_grad(const void* logits, int dtype, long long rows, int vocab, long long row_stride, void* grad,
                                     long long grad_stride, const void* targets, int wide_targets, long long ignore_index, float inv_t, int top,
                                     const float* stats, const float* entropy, const long long* top_tokens, const float* g_log_prob,
                                     const float* g_entropy, const float* g_top, cudaStream_t stream) {
  if (rows <= 0) return 0;
  const long long size = dtype == 0 ? 4 : 2;
  if ((((uintptr_t)logits ^ (uintptr_t)grad) & 15u) != 0 || ((row_stride - grad_stride) * size) % 16 != 0) {
    psgd_set_error("psgd_token_logprob_grad: rows of the gradient do not lie as those of the logits");
    return -1;
  }
  LpGradArgs a = {logits, row_stride, grad, grad_stride, targets, wide_targets, ignore_index, rows, vocab, 1, inv_t, inv_t * (1.f / LP_LN2),
                  g_top ? top : 0, (const float2*)stats, entropy, top_tokens, g_log_prob, g_entropy, g_top};
  if (dtype == 0) return lp_grad_dispatch<float>(a, stream);
  if (dtype == 1) return lp_grad_dispatch<__nv_bfloat16>(a, stream);
  return lp_grad_dispatch<__half>(a, stream);
}
