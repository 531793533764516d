// Attention over packed sequences, causal or not, with grouped heads: forward and backward on the tensor cores.
//
//   S = scale Q K^T (masked),  P = softmax(S),  O = P V
//   delta = rowsum(dO o O),  dP = dO V^T,  dS = P o (dP - delta)
//   dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q
//
// Q, dO and O are [tokens, query heads, size], K and V [tokens, key heads, size]; sequence s has the rows offsets[s] to
// offsets[s + 1], read on the device. Products take 16-bit operands and accumulate in float32; maxima, sums and the
// logarithm of the sum are float32; P and dS are rounded to 16 bits as operands of the second products, as the tensor
// core takes them, and results are rounded once.
//
// Rows of Q, K, V and dO come by TMA, and the scores never leave tensor memory and registers: in the forward pass a thread owns a row of a
// tile (a lane of tensor memory), so that a row's maximum and sum need no exchange between lanes; in the backward pass, which
// needs neither, two threads share it. P and dS go back to tensor memory as the A operand of the second products. A step's chain
// (products, into registers, exponentials, back, products) is much longer than the work of any one unit in it, so two chains run on
// every SM: two blocks, or two tiles of one.
//   forward   tiles of 128 queries, walking over tiles of 128 keys.
//   dQ        tiles of 128 queries, walking over tiles of 64 keys.
//   dK, dV    tiles of 128 keys, walking over tiles of 64 queries of all heads of the group, transposed: lanes are
//             keys, so that P^T and dS^T are A operands as they come. Nothing is added with atomics: the same inputs
//             give the same bits. The price is that S and dP are computed twice (seven products instead of five).
// float16: weights and dS are multiplied with powers of two in the backward pass, so that small ones keep their bits.
// A row of a tile that belongs to another sequence, or lies behind the last one, may hold anything: before it is multiplied with anything
// but scores that are replaced, its row in shared memory is cleared.
//
// Heads of 64, four sequences of 4096: 690 TFLOP/s forward, 570 to 630 backward (counted as five products); heads of 128 1000 to 1080 and 635; GPT-2
// medium's step over documents of 24 to 1024, 49 GFLOP, 38 + 99 us. Bound by the chains: with two of them the tensor cores are 43 to 55 % busy
// in the backward pass, the special functions 51 to 58 % (heads of 64), instructions are issued in 42 to 45 % of all cycles.
//
// Blocks are dealt out with the longest first: the device finds the n-th tile in the order of its distance from the
// sequence's beginning (causal: of its work), from the offsets alone.
//
// Every wait is bounded: where one runs out, the block sets the status word, all its warps fall through, and the
// kernel ends.
#include <cooperative_groups.h>
#include <cuda.h>
#include <string.h>

#include "psgd_umma.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int AT_TILE = 128;     // rows of a tile that stays
constexpr int AT_STEP = 64;      // rows of a tile that passes, in the backward pass
constexpr float AT_LOG2E = 1.44269504088896341f;

struct AtArgs {
  CUtensorMap q, k, v, g;        // boxes of 64 elements x 1 head x 64 rows; g: the gradient of the output
  const int* offsets;
  const int* plan;               // where there are more sequences than a warp has lanes: see below; else null
  int sequences, tokens, heads, group, size;   // group: query heads per key head
  int causal;
  float scale, scale2;           // scale, scale log2(e)
  int split;                     // dK, dV: blocks that share a tile of keys
  int blocks;                    // tiles (forward: pairs of them) that the grid has room for, per head
  const void* out;               // forward: written; backward: read. [tokens, heads, size]
  const void* rest;              // what rounding took from the output, likewise; null where no gradient will be asked for
  const void* grad;              // the gradient of the output, as `g` addresses it
  long long grad_row, grad_head; // its strides
  const void* value;             // V likewise
  long long value_row, value_head;
  int* lengths_v;                // [key heads, tokens], float16: at the first row of each tile an exponent of its longest row of V, see below
  int* lengths_g;                // [heads, tokens], likewise of dO
  float* lse;                    // [heads, tokens]: log2 of the sum of exponentials, scaled scores
  float* delta;                  // [heads, tokens]
  void *dq, *dk, *dv;
  int* status;
};

__device__ __forceinline__ float at_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The largest of three; what is no number wins.
__device__ __forceinline__ float at_max3(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// 2^x in plain arithmetic: x = n + f with |f| <= 1/2 by rounding, a polynomial of degree 4 in f with the least maximal relative error
// (2.8e-6; fitted with value 1 at 0), n added to the exponent. Below -127 the result is zero, and of what is no number it is any: a row that
// holds such a score has a maximum that is none, and the exponentials beside this one say so.
constexpr int AT_POLY = 2;   // of 16 exponentials, those that are taken so: the special function unit has 16 results per cycle and SM
__device__ __forceinline__ float2 at_exp2_poly(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f), back = make_float2(-12582912.f, -12582912.f), minus = make_float2(-1.f, -1.f);
  x.x = fmaxf(x.x, -127.f);
  x.y = fmaxf(x.y, -127.f);
  const float2 t = add2(x, magic);
  const float2 f = fma2(add2(t, back), minus, x);
  float2 p = make_float2(0.0095828531f, 0.0095828531f);
  p = fma2(p, f, make_float2(0.0559064246f, 0.0559064246f));
  p = fma2(p, f, make_float2(0.2402409861f, 0.2402409861f));
  p = fma2(p, f, make_float2(0.6931241934f, 0.6931241934f));
  p = fma2(p, f, make_float2(1.f, 1.f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)), __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}

// ---- which tile --------------------------------------------------------------------------------
// Sequences cut into pieces of `rows`; piece number `index` in the order: the pieces that have the most of their sequence before them
// (`from_end`: behind them) first. One warp asks. Returns false where there are fewer.
struct AtPiece {
  int start, length, piece;      // first row and rows of its sequence, its number there
  int before, behind;            // rows that belong to no sequence: [0, before) and [behind, tokens)
};
__device__ __forceinline__ int at_bound(const int* offsets, int s, int tokens) { return min(max(offsets[s], 0), tokens); }
__device__ bool at_find(const AtArgs& a, int rows, int index, bool from_end, AtPiece& out) {
  const int lane = threadIdx.x & 31;
  if (a.plan != nullptr) {       // the order has been written down: how many there are, then start, length and level of each
    out.before = at_bound(a.offsets, 0, a.tokens);
    out.behind = max(at_bound(a.offsets, a.sequences, a.tokens), out.before);
    if (index >= a.plan[0]) return false;
    const int* x = a.plan + 1 + 3ll * index;
    out.start = x[0];
    out.length = x[1];
    out.piece = from_end ? (out.length + rows - 1) / rows - 1 - x[2] : x[2];
    return true;
  }
  int begin = 0, length = 0;     // of the sequence that this lane has
  if (lane < a.sequences) {
    begin = at_bound(a.offsets, lane, a.tokens);
    length = max(at_bound(a.offsets, lane + 1, a.tokens) - begin, 0);
  }
  const int mine = (length + rows - 1) / rows;
  out.before = at_bound(a.offsets, 0, a.tokens);
  out.behind = max(at_bound(a.offsets, a.sequences, a.tokens), out.before);
  // pieces at level `level` of their sequences or above
  auto above = [&](int level) { return (int)__reduce_add_sync(0xffffffffu, (unsigned)max(mine - level, 0)); };
  if (index >= above(0)) return false;
  int lo = 0, hi = (int)__reduce_max_sync(0xffffffffu, (unsigned)mine);         // above(lo) > index >= above(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (above(mid) > index) lo = mid;
    else hi = mid;
  }
  // the sequence that has more than `lo` pieces as the index says
  const unsigned deep = __ballot_sync(0xffffffffu, mine > lo);
  const int nth = index - above(lo + 1), from = __ffs(__ballot_sync(0xffffffffu, mine > lo && __popc(deep & ((1u << lane) - 1)) == nth)) - 1;
  out.start = __shfl_sync(0xffffffffu, begin, from);
  out.length = __shfl_sync(0xffffffffu, length, from);
  out.piece = from_end ? __shfl_sync(0xffffffffu, mine, from) - 1 - lo : lo;
  return true;
}

// The same order written down, for more sequences than 32: block `level` has the pieces of that level. Their places follow those of all higher levels,
// in the order of their sequences. (A block that asked for itself as above, in turns of 32 sequences, would read all offsets again for every
// question: with thousands of sequences that is more than its work.)
// Counts are of 64 bits: of lists that go down, where long sequences overlap again and again, the pieces may be more than 2^31, of which
// those that the grid has room for are written down.
constexpr int AT_PLAN_THREADS = 256;
__global__ void __launch_bounds__(AT_PLAN_THREADS) psgd_attention_plan_kernel(const int* offsets, int sequences, int tokens, int rows, int capacity, int* plan) {
  __shared__ long long s_wide[AT_PLAN_THREADS / 32];
  __shared__ int s_sum[AT_PLAN_THREADS / 32];
  const int level = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto sum = [&](long long x) {  // over the block
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    __syncthreads();
    if (lane == 0) s_wide[warp] = x;
    __syncthreads();
    long long all = 0;
    for (int w = 0; w < AT_PLAN_THREADS / 32; ++w) all += s_wide[w];
    return all;
  };
  long long higher = 0, here = 0, total = 0;
  for (int s = threadIdx.x; s < sequences; s += AT_PLAN_THREADS) {
    const int n = (max(at_bound(offsets, s + 1, tokens) - at_bound(offsets, s, tokens), 0) + rows - 1) / rows;
    higher += max(n - level - 1, 0);
    here += n > level;
    total += n;
  }
  higher = sum(higher);
  here = sum(here);
  if (level == 0) {
    total = sum(total);
    if (threadIdx.x == 0) plan[0] = (int)min(total, (long long)capacity);
  }
  if (here == 0 || higher >= capacity) return;
  long long at = higher;
  for (int s0 = 0; s0 < sequences && at < capacity; s0 += AT_PLAN_THREADS) {
    const int s = s0 + threadIdx.x;
    int begin = 0, length = 0;
    if (s < sequences) {
      begin = at_bound(offsets, s, tokens);
      length = max(at_bound(offsets, s + 1, tokens) - begin, 0);
    }
    const bool has = (length + rows - 1) / rows > level;
    const unsigned votes = __ballot_sync(0xffffffffu, has);
    __syncthreads();
    if (lane == 0) s_sum[warp] = __popc(votes);
    __syncthreads();
    int before = __popc(votes & ((1u << lane) - 1)), all = 0;
    for (int w = 0; w < AT_PLAN_THREADS / 32; ++w) {
      before += w < warp ? s_sum[w] : 0;
      all += s_sum[w];
    }
    const long long place = at + before;
    if (has && place < capacity) {
      int* x = plan + 1 + 3 * place;
      x[0] = begin;
      x[1] = length;
      x[2] = level;
    }
    at += all;
  }
}

// Rows of a result that belong to no sequence: zeros. Dealt out over the blocks of a head.
template <typename T>
__device__ __forceinline__ void at_clear_outside(const AtArgs& a, const AtPiece& piece, T* out, int heads, int head, int block) {
  const unsigned outside = a.tokens - (piece.behind - piece.before), before = piece.before;      // (a row and a step behind it may pass 2^31)
  for (unsigned i = block; i < outside; i += a.blocks) {
    const int row = (int)(i < before ? i : i + (piece.behind - piece.before));
    T* p = out + ((long long)row * heads + head) * a.size;
    for (int e = threadIdx.x; e < a.size; e += blockDim.x) p[e] = T(0.f);
  }
}

// ---- pieces of the pipelines -------------------------------------------------------------------
// Waits for a whole warp, which goes on as one: all of its lanes, or none. (A lane that gave up alone would leave the others waiting for it at their next
// common instruction.)
struct AtWait {
  volatile int* abort_flag;
  int* status;
  __device__ __forceinline__ bool one(uint64_t* bar, uint32_t parity) const {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)   // (the clock is read only when it takes longer)
      if (psgd_mbar_try_wait(bar, parity)) return true;
    return psgd_mbar_wait(bar, parity, abort_flag, status);
  }
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const { return __all_sync(0xffffffffu, one(bar, parity)); }
};

// One arrival for a warp whose lanes have all done what the barrier stands for.
__device__ __forceinline__ void at_arrive(uint64_t* bar) {
  umma_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) psgd_mbar_arrive(bar);
}

// A tile of ROWS rows from `row` of one head, in boxes of 64 rows x 64 elements.
template <int PANELS, int ROWS>
__device__ __forceinline__ void at_load_tile(uint32_t dst, const CUtensorMap* map, int head, int row, uint64_t* bar) {
#pragma unroll
  for (int p = 0; p < PANELS; ++p) {
#pragma unroll
    for (int r = 0; r < ROWS; r += 64) tma_load_box3(dst + (p * ROWS + r) * 128, map, p * 64, head, row + r, bar);
  }
}

// Clears the rows of a tile from `from` on, which do not belong to the sequence and may hold anything: by the warp that issues the products, before
// it does so.
template <int PANELS, int ROWS>
__device__ __forceinline__ void at_clear_rows(uint8_t* tile, int from) {
#pragma unroll 1
  for (int p = 0; p < PANELS; ++p) {
#pragma unroll 1
    for (int i = from * 8 + (int)(threadIdx.x & 31); i < ROWS * 8; i += 32) reinterpret_cast<uint4*>(tile + p * ROWS * 128)[i] = make_uint4(0, 0, 0, 0);
  }
  psgd_fence_async_shared();
  __syncwarp();
}

// The 32 rows of an accumulator that a warp can read, times `factor`, as rows of 16-bit numbers `pitch` elements apart, the first `rows` of them;
// what rounding takes from them likewise to `rest`. By way of 4 KiB of shared memory of the warp's own: a lane has a row, and eight lanes
// together write 128 bytes of one.
template <typename T, int PANELS>
__device__ __forceinline__ void at_write_rows(uint32_t tmem, float factor, uint8_t* stage, T* out, T* rest, long long pitch, int rows, int size) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int panel = 0; panel < PANELS; ++panel) {
    if (panel * 64 >= size) break;
    float f[64];
    tmem_load32(tmem + panel * 64, f);
    tmem_load32(tmem + panel * 64 + 32, f + 32);
    tmem_load_wait<64>(f);
#pragma unroll
    for (int c = 0; c < 64; ++c) f[c] *= factor;
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
      T* to = part == 0 ? out : rest;
      if (to == nullptr) break;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float& x = f[8 * c + 2 * e];
          float& y = f[8 * c + 2 * e + 1];
          w[e] = pack2<T>(x, y);
          const float2 back = unpack2<T>(w[e]);
          x -= back.x;
          y -= back.y;
        }
        *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = i * 4 + (lane >> 3), c = lane & 7;
        const uint4 v = *reinterpret_cast<const uint4*>(stage + row * 128 + ((c ^ (row & 7)) << 4));
        if (row < rows && panel * 64 + c * 8 < size) *reinterpret_cast<uint4*>(to + row * pitch + panel * 64 + c * 8) = v;
      }
      __syncwarp();
    }
  }
}

template <typename T>
struct AtType;   // as the instruction descriptor names it
template <>
struct AtType<__half> { static constexpr int value = 0; };
template <>
struct AtType<__nv_bfloat16> { static constexpr int value = 1; };

// ---- forward -----------------------------------------------------------------------------------
// TILES of queries per block: four warps each, then a warp that loads and one that issues the products.
constexpr int AF_RING = 4;        // tiles of K and V under way

__host__ __device__ constexpr int af_threads(int tiles) { return 128 * tiles + 64; }
constexpr size_t af_shared(int panels, int tiles) { return 1024 + (size_t)(tiles + AF_RING) * panels * UMMA_PANEL; }

template <typename T, int PANELS, int TILES>
__global__ void __launch_bounds__(af_threads(TILES), 3 - TILES) psgd_attention_kernel(const __grid_constant__ AtArgs a) {
  constexpr int TILE_BYTES = PANELS * UMMA_PANEL;
  constexpr int LOADER = 4 * TILES, ISSUER = LOADER + 1, COLUMNS = 256 * TILES, O = TILES * AT_TILE;   // warps; tensor memory: scores, outputs
  // Where there is room P has columns of its own, and the next scores are multiplied as soon as these are in registers; else P takes the place
  // of the scores, and the next ones come behind P V.
  constexpr bool EARLY = TILES == 1 && PANELS == 1;
  constexpr int P = EARLY ? 192 : 0;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = base;
  uint8_t* s_ring = base + TILES * TILE_BYTES;
  __shared__ __align__(8) uint64_t bar_q, bar_full[AF_RING], bar_empty[AF_RING], bar_s[TILES], bar_r[TILES], bar_p[TILES][2], bar_o[TILES];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_found;
  __shared__ AtPiece s_piece;

  const int tid = threadIdx.x, warp = warp_uniform(tid >> 5), lane = tid & 31;
  const int head = blockIdx.x % a.heads, index = blockIdx.x / a.heads;
  if (warp == 0) {
    AtPiece piece = {0, 0, 0, 0, 0};
    const bool found = at_find(a, TILES * AT_TILE, index, false, piece);
    if (lane == 0) {
      s_piece = piece;
      s_found = found;
    }
  }
  if (warp == LOADER && lane < 3) tma_prefetch_map(lane == 0 ? &a.q : lane == 1 ? &a.k : &a.v);
  if (tid == 32) {
    psgd_mbar_init(&bar_q, 1);
    for (int i = 0; i < AF_RING; ++i) {
      psgd_mbar_init(&bar_full[i], 1);
      psgd_mbar_init(&bar_empty[i], 1);
    }
    for (int t = 0; t < TILES; ++t) {
      psgd_mbar_init(&bar_s[t], 1);
      psgd_mbar_init(&bar_r[t], 4);
      psgd_mbar_init(&bar_p[t][0], 4);
      psgd_mbar_init(&bar_p[t][1], 4);
      psgd_mbar_init(&bar_o[t], 1);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ISSUER) tmem_alloc(&s_tmem, COLUMNS);
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  at_clear_outside<T>(a, s_piece, (T*)a.out, a.heads, head, index);
  if (!s_found) {
    if (warp == ISSUER) tmem_free(s_tmem, COLUMNS);
    return;
  }
  const uint32_t tmem = warp_uniform(s_tmem);
  const AtWait wait = {&s_abort, a.status};
  const int start = s_piece.start, length = warp_uniform(s_piece.length), row0 = warp_uniform(s_piece.piece) * TILES * AT_TILE;
  // tiles of keys that each tile of queries meets
  int n[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const int q0 = row0 + t * AT_TILE;
    n[t] = q0 >= length ? 0 : a.causal ? q0 / AT_TILE + 1 : (length + AT_TILE - 1) / AT_TILE;
  }
  const int steps = max(n[0], n[TILES - 1]);

  if (warp == LOADER) {
    {
      if (lane == 0) psgd_mbar_expect_tx(&bar_q, n[TILES - 1] > 0 ? TILES * TILE_BYTES : TILE_BYTES);
      for (int t = 0; t < TILES; ++t)
        if (n[t] > 0 && lane == 0) at_load_tile<PANELS, AT_TILE>(psgd_smem_u32(s_q + t * TILE_BYTES), &a.q, head, start + row0 + t * AT_TILE, &bar_q);
      for (int i = 0; i < 2 * steps; ++i) {   // K_0, V_0, K_1, V_1, ...
        const int slot = i % AF_RING;
        if (!wait(&bar_empty[slot], ((i / AF_RING) & 1) ^ 1)) break;
        if (lane != 0) continue;
        psgd_mbar_expect_tx(&bar_full[slot], TILE_BYTES);
        at_load_tile<PANELS, AT_TILE>(psgd_smem_u32(s_ring + slot * TILE_BYTES), (i & 1) ? &a.v : &a.k, head / a.group, start + (i >> 1) * AT_TILE, &bar_full[slot]);
      }
    }
  } else if (warp == ISSUER) {
    const int k_steps = (a.size + 15) / 16;
    constexpr uint32_t S_SHAPE = umma_shape(AtType<T>::value, false, AT_TILE);
    const uint32_t o_shape = umma_shape(AtType<T>::value, true, k_steps * 16);
    const uint32_t q_at = warp_uniform(psgd_smem_u32(s_q)), ring_at = q_at + TILES * TILE_BYTES;
    bool ok = wait(&bar_q, 0) && wait(&bar_full[0], 0);
    int have = 0;   // tiles of keys that are there
    auto scores = [&](int t, int j) {
      if (j > have) {
        ok = wait(&bar_full[2 * j % AF_RING], (2 * j / AF_RING) & 1);
        have = j;
      }
      if (!ok) return;
      umma_fence_after();
      umma_rows_by_rows<4 * PANELS, AT_TILE>(tmem + t * AT_TILE, q_at + t * TILE_BYTES, ring_at + (2 * j % AF_RING) * TILE_BYTES, S_SHAPE, k_steps);
      umma_arrive(&bar_s[t]);
    };
    for (int t = 0; t < TILES && ok; ++t)
      if (n[t] > 0) scores(t, 0);
    if (ok) umma_arrive(&bar_empty[0]);
    for (int j = 0; j < steps && ok; ++j) {
      const int kv = 2 * j + 1, kn = 2 * j + 2;
      for (int t = 0; t < TILES && ok; ++t) {
        if (j >= n[t]) continue;
        if (EARLY && j + 1 < n[t]) {
          ok = wait(&bar_r[t], j & 1);
          if (ok) scores(t, j + 1);
          if (!ok) break;
        }
        if (t == 0 || n[0] <= j) {
          ok = wait(&bar_full[kv % AF_RING], (kv / AF_RING) & 1);
          if (ok && length - j * AT_TILE < AT_TILE) at_clear_rows<PANELS, AT_TILE>(s_ring + (kv % AF_RING) * TILE_BYTES, length - j * AT_TILE);
        }
        const uint32_t o_at = tmem + O + t * AT_TILE, p_at = tmem + P + t * AT_TILE, v_at = ring_at + (kv % AF_RING) * TILE_BYTES;
        ok = ok && wait(&bar_p[t][0], j & 1);
        if (!ok) break;
        umma_fence_after();
        umma_weights_by_rows<0, 4, AT_TILE>(o_at, p_at, v_at, o_shape, j > 0);
        ok = wait(&bar_p[t][1], j & 1);
        if (!ok) break;
        umma_fence_after();
        umma_weights_by_rows<4, 8, AT_TILE>(o_at, p_at, v_at, o_shape, true);
        umma_arrive(&bar_o[t]);
        if (!EARLY && j + 1 < n[t]) scores(t, j + 1);
      }
      if (!ok) break;
      umma_arrive(&bar_empty[kv % AF_RING]);
      if (j + 1 < steps) umma_arrive(&bar_empty[kn % AF_RING]);
    }
  } else {
    const int t = warp >> 2, row = tid & 127;
    const int q = row0 + t * AT_TILE + row;          // in its sequence
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * AT_TILE, o_at = tmem + lanes + O + t * AT_TILE, p_at = tmem + lanes + P + t * AT_TILE;
    const int limit = a.causal ? min(q, length - 1) : length - 1;   // last key that counts
    float m = -INFINITY, l = 0.f;                    // what exponents are relative to (unscaled scores), sum
    bool ok = true;
    for (int j = 0; j < n[t]; ++j) {
      ok = wait(&bar_s[t], j & 1);
      if (!ok) break;
      umma_fence_after();
      float s[AT_TILE];
#pragma unroll
      for (int c = 0; c < AT_TILE; c += 32) tmem_load32(s_at + c, s + c);
      tmem_load_wait<AT_TILE>(s);
      if (EARLY) at_arrive(&bar_r[t]);
      if (j == n[t] - 1) {
        const int last = limit - j * AT_TILE;
#pragma unroll
        for (int c = 0; c < AT_TILE; ++c)
          if (c > last) s[c] = -INFINITY;
      }
      float most[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) most[c] = at_max3(s[c], s[c + 4], s[c + 8]);
#pragma unroll
      for (int c = 12; c < AT_TILE - 4; c += 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) most[i] = at_max3(most[i], s[c + i], s[c + i + 4]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) most[i] = at_max3(most[i], s[AT_TILE - 4 + i], s[AT_TILE - 4 + i]);
      const float largest = at_max3(at_max3(most[0], most[1], most[2]), most[3], most[3]);
      if (j == 0) {
        m = largest;
      } else {
        // The sums stay relative to an older maximum while exponents stay below 2^8: accumulators are rescaled only when it moves by
        // more (and where it is no number; not where all scores so far are -inf, which are no distance apart).
        const bool moves = !((largest - m) * a.scale2 <= 8.f) && largest != -INFINITY;
        if (__any_sync(0xffffffffu, moves)) {
          ok = wait(&bar_o[t], (j - 1) & 1);
          if (!ok) break;
          umma_fence_after();
          const float f = moves ? at_exp2((m - largest) * a.scale2) : 1.f;
          if (moves) m = largest;
          l *= f;
#pragma unroll
          for (int c = 0; c < PANELS * 64; c += 32) {
            if (c >= a.size) break;
            float o[32];
            tmem_load32(o_at + c, o);
            tmem_load_wait<32>(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= f;
            tmem_store16(o_at + c, reinterpret_cast<uint32_t*>(o));
            tmem_store16(o_at + c + 16, reinterpret_cast<uint32_t*>(o) + 16);
          }
        }
      }
      const float from = m == -INFINITY ? 0.f : m * a.scale2;
      const float2 factor2 = make_float2(a.scale2, a.scale2), from2 = make_float2(-from, -from);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int c = half * 64; c < half * 64 + 64; c += 32) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 x = fma2(make_float2(s[c + i], s[c + i + 1]), factor2, from2);
            const float2 e = i % 16 < AT_POLY ? at_exp2_poly(x) : make_float2(at_exp2(x.x), at_exp2(x.y));
            sum[(i / 2) & 1] = add2(sum[(i / 2) & 1], e);
            p[i / 2] = pack2<T>(e.x, e.y);
          }
          if (EARLY && c == 0 && j > 0) {
            ok = wait(&bar_o[t], (j - 1) & 1);   // the last P has been read
            umma_fence_after();
          }
          tmem_store16(p_at + c / 2, p);
        }
        tmem_store_wait();
        at_arrive(&bar_p[t][half]);
      }
      if (!ok) break;
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    }
    if (ok && n[t] > 0) ok = wait(&bar_o[t], (n[t] - 1) & 1);
    if (ok && n[t] > 0) {
      umma_fence_after();
      const int first = row0 + t * AT_TILE + (warp & 3) * 32;      // the warp's rows
      const long long at = ((long long)(start + first) * a.heads + head) * a.size;
      at_write_rows<T, PANELS>(o_at, 1.f / l, s_q + t * TILE_BYTES + (warp & 3) * 4096, (T*)a.out + at, a.rest == nullptr ? nullptr : (T*)a.rest + at,
                               (long long)a.heads * a.size, length - first, a.size);
      if (q < length) a.lse[(long long)head * a.tokens + start + q] = m * a.scale2 + log2f(l);
    }
  }
  umma_fence_before();
  __syncthreads();
  if (s_abort) {
    psgd_let_copies_land();
    __syncthreads();
  }
  if (warp == ISSUER) {
    __syncwarp();
    tmem_free(tmem, COLUMNS);
  }
}

// ---- backward ----------------------------------------------------------------------------------
constexpr int AB_MOST_SPLIT = 8;      // blocks of a cluster
constexpr int AB_ENOUGH = 4 * 148;    // with so many blocks the heads of a group stay in one
// CHAINS of eight warps each take the steps in turn; then a warp that loads and one that issues the products. One chain where two blocks fit an SM,
// two where one does. Two threads share a row of a tile, AB_WIDE columns each.
__host__ __device__ constexpr int ab_threads(int chains) { return 256 * chains + 64; }
constexpr int AB_WIDE = AT_STEP / 2;
constexpr int AB_GAP = AB_WIDE / 2;   // columns: each thread's 16-bit numbers take the first half of its own place
// In sequences up to this long dS goes into the products in two parts, what rounding took from it in the second half of its place. Few terms leave more of
// their roundings in a sum: dQ and dK were 1.45 to 1.54 times as far from 64 bits as results that are only rounded, 1.05 to 1.15 times so. (Longer
// sequences: 1.45. There the second products would cost 10 to 20 %: documents of 24 to 1024 forward and backward 137.7 / 147.1 us, 4 x 4096
// heads of 128 backward 1080 / 1310; here they are not seen, 7 sequences up to 64 15.7 / 15.8.)
constexpr int AB_FINE = AT_TILE;
// Tiles that pass come in pairs (K and V, or Q and dO).
__host__ __device__ constexpr int ab_stages(int panels) { return panels == 1 ? 3 : 4; }
constexpr int AB_ONES = 2 * AT_TILE * 16, AB_STATS = 2 * 2 * AT_STEP * 16;   // bytes: rows of 16 elements, see umma_add_columns
// `more`: bytes besides the tiles.
__host__ __device__ constexpr size_t ab_shared(int panels, int more) { return 1024 + (size_t)panels * (2 + ab_stages(panels)) * UMMA_PANEL + more; }

template <int CHAINS, int STAGES>
struct AbBars {
  uint64_t fixed, full[STAGES], empty[STAGES], s[CHAINS], dp[CHAINS], p[CHAINS], ds[CHAINS], done;
  __device__ __forceinline__ void init(int of_fixed, int of_full) {
    psgd_mbar_init(&fixed, of_fixed);
    for (int i = 0; i < STAGES; ++i) {
      psgd_mbar_init(&full[i], of_full);
      psgd_mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < CHAINS; ++i) {
      psgd_mbar_init(&s[i], 1);
      psgd_mbar_init(&dp[i], 1);
      psgd_mbar_init(&p[i], 8);
      psgd_mbar_init(&ds[i], 8);
    }
    psgd_mbar_init(&done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
};

// Exponentials 2^(scale2 s - at) of a row.
__device__ __forceinline__ void ab_exponentials(float* s, float scale2, float at) {
  const float2 factor = make_float2(scale2, scale2), minus = make_float2(-at, -at);
#pragma unroll
  for (int c = 0; c < AB_WIDE; c += 2) {
    const float2 x = fma2(make_float2(s[c], s[c + 1]), factor, minus);
    s[c] = at_exp2(x.x);
    s[c + 1] = at_exp2(x.y);
  }
}

// What rounding took from `x`, as rounded in `w`.
template <typename T>
__device__ __forceinline__ void ab_store_rest(uint32_t at, const float* x, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < AB_WIDE; i += 2) {
    const float2 back = unpack2<T>(w[i / 2]);
    w[i / 2] = pack2<T>(x[i] - back.x, x[i + 1] - back.y);
  }
  tmem_store16(at, w);
}

// Powers of two, float16. dS is small wherever gradients are: a weight of 1 / 4096 and a gradient of 2^-10 make 2^-19, of which float16, whose normal
// numbers end at 2^-14, holds five bits. So dS is multiplied with a power of two before it is rounded, which the last scaling takes back:
//   |dS| <= |P| (|dP| + |delta|) <= 2 |dO_i| max_j |V_j|,
// and the largest power is taken that keeps this below 2^14. In dQ each row has its own; dK sums over rows, which share that of the longest dO
// of all that see the tile's keys. (One power for all inputs would have to keep the largest gradients finite.) It rides on operations that
// are there: in dQ a sum becomes a fused one; in dK, dV it is added to exponents, so that the weights have it too. Those are small in long
// sequences, 1 / length as a rule: their power is at least the one that brings this to 2^-10, and where it is above that of dS what dS is made of
// is multiplied with the difference. Rows of what is no number have no say: whatever they touch is none either. bfloat16 has the
// range of float32 and needs none of this.
template <typename T>
constexpr bool AB_SHIFTS = AtType<T>::value == 0;
constexpr int AB_ROOM = 13;           // 2^(shift + exponents of both lengths + 1) <= 2^14
constexpr int AB_MOST_SHIFT = 14;     // (weights times 2^14 are finite, and a scale of 2^-100 times 2^-14 is a normal number)
// The least e for which a vector is shorter than 2^e, from the square of its length; of what is not finite as of zeros.
__device__ __forceinline__ int ab_exponent(float square) {
  const int b = (int)(__float_as_uint(square) >> 23 & 0xFF);
  return b == 0xFF ? -63 : (b - 125) >> 1;
}
__device__ __forceinline__ float ab_power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ int ab_lift(int shift, int length) { return max(max(shift, 0), min(22 - __clz(length), AB_MOST_SHIFT)); }   // of P
__device__ __forceinline__ float ab_square(uint4 x, float square) {   // (of eight float16)
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack2<__half>(w[j]);
    square = fmaf(f.x, f.x, fmaf(f.y, f.y, square));
  }
  return square;
}
// What the longest rows of V leave of AB_ROOM, and where asked those of dO of the heads that share them, in the tiles from `from` on. A warp asks.
__device__ __forceinline__ int ab_room(const AtArgs& a, int kv_head, int start, int length, bool gradients, int from) {
  const int tiles = (length + AT_TILE - 1) / AT_TILE, heads = gradients ? a.group : 0;
  const int* v = a.lengths_v + (long long)kv_head * a.tokens + start;
  const int* g = a.lengths_g + (long long)kv_head * a.group * a.tokens + start;
  int of_v = -63, of_g = -63;
  for (int i = (int)(threadIdx.x & 31); i < tiles; i += 32) {
    const int at = i * AT_TILE;
    of_v = max(of_v, v[at]);
    if (i < from) continue;
#pragma unroll 4
    for (int h = 0; h < heads; ++h) of_g = max(of_g, g[(long long)h * a.tokens + at]);
  }
  of_v = __reduce_max_sync(0xffffffffu, of_v);
  return AB_ROOM - of_v - (gradients ? __reduce_max_sync(0xffffffffu, of_g) : 0);
}

// Exponents of the rows of V; those of dO come from the pass over the queries, which begins beside this one. (3357 rows of 4 heads of 80: 3.5 us, of which
// 2.3 are seen; the whole of it, with the weights' powers, takes 131 to 135 us of forward and backward pass.)
constexpr int AN_THREADS = 256;
__global__ void __launch_bounds__(AN_THREADS) psgd_attention_lengths_kernel(const __grid_constant__ AtArgs a) {
  __shared__ int s_most[AN_THREADS / 32], s_found;
  __shared__ AtPiece s_piece;
  psgd_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, kv_heads = a.heads / a.group;
  const int head = blockIdx.x % kv_heads, index = blockIdx.x / kv_heads;
  if (tid < 32) {
    AtPiece piece = {0, 0, 0, 0, 0};
    const bool found = at_find(a, AT_TILE, index, false, piece);
    if (lane == 0) {
      s_piece = piece;
      s_found = found;
    }
  }
  __syncthreads();
  if (!s_found) return;
  constexpr int LOADS = AT_TILE / (AN_THREADS / 16);       // 16 lanes to a row
  const long long row0 = s_piece.start + (long long)s_piece.piece * AT_TILE;
  const int rows = min(AT_TILE, s_piece.length - s_piece.piece * AT_TILE), c = tid % 16 * 8;
  const __half* v = (const __half*)a.value + head * a.value_head + row0 * a.value_row + c;
  uint4 x[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int r = tid / 16 + i * (AN_THREADS / 16);
    x[i] = make_uint4(0, 0, 0, 0);
    if (r < rows && c < a.size) x[i] = *reinterpret_cast<const uint4*>(v + r * a.value_row);
  }
  int e = -63;
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    float square = ab_square(x[i], 0.f);
#pragma unroll
    for (int by = 8; by > 0; by >>= 1) square += __shfl_xor_sync(0xffffffffu, square, by);
    e = max(e, ab_exponent(square));
  }
  e = __reduce_max_sync(0xffffffffu, e);
  if (lane == 0) s_most[tid / 32] = e;
  __syncthreads();
  if (tid != 0) return;
  for (int w = 1; w < AN_THREADS / 32; ++w) e = max(e, s_most[w]);
  a.lengths_v[(long long)head * a.tokens + row0] = e;
}

// dQ: tensor memory holds, per chain, S and dP (64 columns each; dS takes the first half of dP's place), and dQ. S of a chain's next step is
// multiplied as soon as this one is in registers, its dP behind dQ of this one.
template <typename T, int PANELS>
__global__ void __launch_bounds__(ab_threads(PANELS), 3 - PANELS) psgd_attention_dq_kernel(const __grid_constant__ AtArgs a) {
  constexpr int TILE_BYTES = PANELS * UMMA_PANEL, HALF = TILE_BYTES / 2, CHAINS = PANELS, STAGES = ab_stages(PANELS);
  constexpr int DQ = 2 * AT_STEP * CHAINS, COLUMNS = 256 * CHAINS;   // tensor memory; chain c has its scores at 128 c, slopes behind
  constexpr int LOADER = 8 * CHAINS, ISSUER = LOADER + 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = base;
  uint8_t* s_g = base + TILE_BYTES;
  uint8_t* s_ring = base + 2 * TILE_BYTES;   // stage: K, V
  __shared__ __align__(8) AbBars<CHAINS, STAGES> bars;
  __shared__ float s_delta[AT_TILE];
  __shared__ int s_exponent[AB_SHIFTS<T> ? AT_TILE : 1], s_room;      // float16: of the rows of dO; AB_ROOM without the longest row of V
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_found;
  __shared__ AtPiece s_piece;

  const int tid = threadIdx.x, warp = warp_uniform(tid >> 5), lane = tid & 31;
  const int head = blockIdx.x % a.heads, index = blockIdx.x / a.heads;
  psgd_launch_dependents();      // (the pass over the keys begins beside the end of this one)
  if (warp == 0) {
    AtPiece piece = {0, 0, 0, 0, 0};
    const bool found = at_find(a, AT_TILE, index, false, piece);
    if (lane == 0) {
      s_piece = piece;
      s_found = found;
    }
  }
  if (warp == LOADER && lane < 4) tma_prefetch_map(lane == 0 ? &a.q : lane == 1 ? &a.g : lane == 2 ? &a.k : &a.v);
  if (tid == 32) {
    bars.init(1, 1);
    s_abort = 0;
  }
  if (warp == ISSUER) tmem_alloc(&s_tmem, COLUMNS);
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  at_clear_outside<T>(a, s_piece, (T*)a.dq, a.heads, head, index);
  if (!s_found) {
    if (AB_SHIFTS<T>) psgd_wait_for_predecessor();
    if (warp == ISSUER) tmem_free(s_tmem, COLUMNS);
    return;
  }
  const uint32_t tmem = warp_uniform(s_tmem);
  const AtWait wait = {&s_abort, a.status};
  const int start = s_piece.start, length = warp_uniform(s_piece.length), q0 = warp_uniform(s_piece.piece) * AT_TILE;
  const int steps = (a.causal ? min(q0 + AT_TILE, length) + AT_STEP - 1 : length + AT_STEP - 1) / AT_STEP;

  if (warp == LOADER) {
    {
      if (lane == 0) psgd_mbar_expect_tx(&bars.fixed, 2 * TILE_BYTES);
      if (lane == 0) {
        at_load_tile<PANELS, AT_TILE>(psgd_smem_u32(s_q), &a.q, head, start + q0, &bars.fixed);
        at_load_tile<PANELS, AT_TILE>(psgd_smem_u32(s_g), &a.g, head, start + q0, &bars.fixed);
      }
      for (int j = 0; j < steps; ++j) {
        const int slot = j % STAGES;
        if (!wait(&bars.empty[slot], ((j / STAGES) & 1) ^ 1)) break;
        if (lane == 0) {
          psgd_mbar_expect_tx(&bars.full[slot], 2 * HALF);
          const uint32_t at = psgd_smem_u32(s_ring + slot * TILE_BYTES);
          at_load_tile<PANELS, AT_STEP>(at, &a.k, head / a.group, start + j * AT_STEP, &bars.full[slot]);
          at_load_tile<PANELS, AT_STEP>(at + HALF, &a.v, head / a.group, start + j * AT_STEP, &bars.full[slot]);
        }
        if (AB_SHIFTS<T> && j == min(STAGES, steps) - 1) {   // nothing has been waited for yet
          psgd_wait_for_predecessor();
          const int room = ab_room(a, head / a.group, start, length, false, 0);
          if (lane == 0) s_room = room;
          __syncwarp();
          asm volatile("bar.arrive 1, %0;" ::"n"(256 * CHAINS + 32) : "memory");
        }
      }
    }
  } else if (warp == ISSUER) {
    const int k_steps = (a.size + 15) / 16;
    constexpr uint32_t S_SHAPE = umma_shape(AtType<T>::value, false, AT_STEP);
    const uint32_t q_shape = umma_shape(AtType<T>::value, true, k_steps * 16);
    const uint32_t q_at = warp_uniform(psgd_smem_u32(s_q)), g_at = q_at + TILE_BYTES, ring_at = q_at + 2 * TILE_BYTES;
    bool ok = wait(&bars.fixed, 0);
    int have = -1;
    auto there = [&](int j) {
      if (j > have) {
        ok = ok && wait(&bars.full[j % STAGES], (j / STAGES) & 1);
        have = j;
        if (ok && length - j * AT_STEP < AT_STEP) {
          at_clear_rows<PANELS, AT_STEP>(s_ring + j % STAGES * TILE_BYTES, length - j * AT_STEP);
          at_clear_rows<PANELS, AT_STEP>(s_ring + j % STAGES * TILE_BYTES + HALF, length - j * AT_STEP);
        }
      }
      if (ok) umma_fence_after();
      return ok;
    };
    auto scores = [&](int j) {
      if (!there(j)) return;
      umma_rows_by_rows<4 * PANELS, AT_STEP>(tmem + j % CHAINS * 128, q_at, ring_at + j % STAGES * TILE_BYTES, S_SHAPE, k_steps);
      umma_arrive(&bars.s[j % CHAINS]);
    };
    auto slopes = [&](int j) {
      if (!there(j)) return;
      umma_rows_by_rows<4 * PANELS, AT_STEP>(tmem + j % CHAINS * 128 + AT_STEP, g_at, ring_at + j % STAGES * TILE_BYTES + HALF, S_SHAPE, k_steps);
      umma_arrive(&bars.dp[j % CHAINS]);
    };
    for (int j = 0; j < CHAINS && j < steps && ok; ++j) {
      scores(j);
      if (ok) slopes(j);
    }
    for (int j = 0; j < steps && ok; ++j) {
      const int chain = j % CHAINS;
      const uint32_t parity = (j / CHAINS) & 1;
      ok = wait(&bars.p[chain], parity);    // S is in registers
      if (!ok) break;
      umma_fence_after();
      if (j + CHAINS < steps) scores(j + CHAINS);
      ok = ok && wait(&bars.ds[chain], parity);
      if (!ok) break;
      umma_fence_after();
      umma_weights_by_rows<0, 4, AT_STEP, AB_GAP>(tmem + DQ, tmem + chain * 128 + AT_STEP, ring_at + j % STAGES * TILE_BYTES, q_shape, j > 0);
      if (length <= AB_FINE) umma_weights_by_rows<0, 4, AT_STEP, AB_GAP>(tmem + DQ, tmem + chain * 128 + AT_STEP + AB_GAP, ring_at + j % STAGES * TILE_BYTES, q_shape, true);
      umma_arrive(&bars.empty[j % STAGES]);
      if (j + CHAINS < steps) slopes(j + CHAINS);
      if (j == steps - 1) umma_arrive(&bars.done);
    }
  } else {
    const int chain = warp >> 3, half = (warp >> 2) & 1, row = tid & 127, q = q0 + row;
    const bool held = q < length;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = tmem + lanes + chain * 128 + half * AB_WIDE, dp_at = s_at + AT_STEP;
    const long long stat = (long long)head * a.tokens + start + q;
    // delta of the rows, for the keys' pass too. It is a small difference of large sums, and what it is off by moves a whole row of
    // dS one way: it takes the output unrounded, in two parts. (With the rounded one dQ and dK were off by 1.7 times their own
    // rounding, so by 1.4.) Eight lanes to a row of 64: a row to a thread took 5000 cycles, since every load touched 32 lines.
    const float lse = held ? a.lse[stat] : 0.f;
    {
      constexpr int ROWS = AT_TILE / (8 * CHAINS), LOADS = ROWS / 4 * PANELS;    // rows of a warp
      uint4 x[LOADS], y[LOADS], z[LOADS];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {    // all on their way before the first is used
        const int r = warp * ROWS + i / PANELS * 4 + (lane >> 3), c = i % PANELS * 64 + (lane & 7) * 8;
        const bool in = q0 + r < length && c < a.size;
        const long long at = ((long long)(start + q0 + r) * a.heads + head) * a.size + c;
        x[i] = y[i] = z[i] = make_uint4(0, 0, 0, 0);
        if (in) x[i] = *reinterpret_cast<const uint4*>((const T*)a.out + at);
        if (in) y[i] = *reinterpret_cast<const uint4*>((const T*)a.grad + (long long)(start + q0 + r) * a.grad_row + (long long)head * a.grad_head + c);
        if (in) z[i] = *reinterpret_cast<const uint4*>((const T*)a.rest + at);
      }
      float sums[ROWS / 4], squares[ROWS / 4];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, ys[4] = {y[i].x, y[i].y, y[i].z, y[i].w}, zs[4] = {z[i].x, z[i].y, z[i].z, z[i].w};
        if (i % PANELS == 0) sums[i / PANELS] = squares[i / PANELS] = 0.f;
        if (AB_SHIFTS<T>) squares[i / PANELS] = ab_square(y[i], squares[i / PANELS]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 u = unpack2<T>(xs[e]), v = unpack2<T>(ys[e]), w = unpack2<T>(zs[e]);
          sums[i / PANELS] = fmaf(u.x + w.x, v.x, sums[i / PANELS]);
          sums[i / PANELS] = fmaf(u.y + w.y, v.y, sums[i / PANELS]);
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS / 4; ++i) {
#pragma unroll
        for (int by = 4; by > 0; by >>= 1) sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], by);
        if ((lane & 7) == 0) s_delta[warp * ROWS + i * 4 + (lane >> 3)] = sums[i];
        if (AB_SHIFTS<T>) {
#pragma unroll
          for (int by = 4; by > 0; by >>= 1) squares[i] += __shfl_xor_sync(0xffffffffu, squares[i], by);
          if ((lane & 7) == 0) s_exponent[warp * ROWS + i * 4 + (lane >> 3)] = ab_exponent(squares[i]);
        }
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(256 * CHAINS + (AB_SHIFTS<T> ? 32 : 0)) : "memory");
    const float delta = s_delta[row], power = AB_SHIFTS<T> ? ab_power(min(s_room - s_exponent[row], AB_MOST_SHIFT)) : 1.f;
    if (AB_SHIFTS<T> && warp == 0) {
      const int e = __reduce_max_sync(0xffffffffu, max(max(s_exponent[lane], s_exponent[lane + 32]), max(s_exponent[lane + 64], s_exponent[lane + 96])));
      if (lane == 0) a.lengths_g[(long long)head * a.tokens + start + q0] = e;
    }
    if (held && warp < 4) a.delta[stat] = delta;
    const int limit = (a.causal ? q : length - 1) - half * AB_WIDE;    // last key that counts, from this thread's first on
    bool ok = true;
    for (int j = chain; j < steps; j += CHAINS) {
      const uint32_t parity = (j / CHAINS) & 1;
      ok = wait(&bars.s[chain], parity);
      if (!ok) break;
      umma_fence_after();
      float p[AB_WIDE];
      tmem_load32(s_at, p);
      tmem_load_wait<AB_WIDE>(p);
      at_arrive(&bars.p[chain]);
      ab_exponentials(p, a.scale2, lse);
      if ((j + 1) * AT_STEP > (a.causal ? q0 + 1 : length)) {     // some keys do not count for some rows
        const int last = limit - j * AT_STEP;
#pragma unroll
        for (int c = 0; c < AB_WIDE; ++c)
          if (c > last) p[c] = 0.f;
      }
      ok = wait(&bars.dp[chain], parity);
      if (!ok) break;
      umma_fence_after();
      const float2 times = make_float2(power, power), minus = make_float2(-delta * power, -delta * power);
      float d[AB_WIDE];
      tmem_load32(dp_at, d);
      tmem_load_wait<AB_WIDE>(d);
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < AB_WIDE; i += 2) {
        const float2 slope = make_float2(d[i], d[i + 1]);
        const float2 x = mul2(make_float2(p[i], p[i + 1]), AB_SHIFTS<T> ? fma2(slope, times, minus) : add2(slope, minus));
        w[i / 2] = pack2<T>(x.x, x.y);
        d[i] = x.x;
        d[i + 1] = x.y;
      }
      tmem_store16(dp_at, w);
      if (length <= AB_FINE) ab_store_rest<T>(dp_at + AB_GAP, d, w);
      tmem_store_wait();
      at_arrive(&bars.ds[chain]);
    }
    if (ok) ok = wait(&bars.done, 0);
    if (ok) {
      umma_fence_after();
      const int first = q0 + (warp & 3) * 32, panel = CHAINS == 2 ? half : 0;     // heads of more than 64: half of them each
      if (chain == 0 && half < PANELS)
        at_write_rows<T, 1>(tmem + lanes + DQ + panel * 64, a.scale / power, s_q + (panel * 4 + (warp & 3)) * 4096,
                            (T*)a.dq + ((long long)(start + first) * a.heads + head) * a.size + panel * 64, (T*)nullptr, (long long)a.heads * a.size, length - first,
                            a.size - panel * 64);
    }
  }
  umma_fence_before();
  __syncthreads();
  if (s_abort) {
    psgd_let_copies_land();
    __syncthreads();
  }
  if (warp == ISSUER) {
    __syncwarp();
    tmem_free(tmem, COLUMNS);
  }
}

// dK, dV: tensor memory holds, per chain, S^T (P^T takes the first half of its place) and dP^T (dS^T likewise), 64 columns each, and dV and dK. dV
// of a step and S^T of the chain's next are multiplied while dS^T is formed, dK and the next dP^T while the next exponentials are
// taken. Where few tiles of keys share many query heads, the heads are dealt out over a cluster of blocks (`split`), whose sums are
// added in shared memory, in the order of their rank.
// What is subtracted from a column of S^T and dP^T, the logarithm of its sum and its delta, is a 32-bit number in three parts of eight bits: one more
// step of the products, with ones. (As numbers that every thread reads they took more of shared memory's time than all operands
// together, since a row of threads reads one word at a time.)
template <typename T, int PANELS>
__global__ void __launch_bounds__(ab_threads(PANELS), 3 - PANELS) psgd_attention_dkv_kernel(const __grid_constant__ AtArgs a) {
  constexpr int CHAINS = PANELS;
  constexpr int TILE_BYTES = PANELS * UMMA_PANEL, HALF = TILE_BYTES / 2, STAGES = ab_stages(PANELS);
  constexpr int DV = 2 * AT_STEP * CHAINS, DK = DV + 64 * PANELS, COLUMNS = 256 * CHAINS;   // tensor memory; chain c has its scores at 128 c, slopes behind
  constexpr int LOADER = 8 * CHAINS, ISSUER = LOADER + 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_k = base;
  uint8_t* s_v = base + TILE_BYTES;
  uint8_t* s_ring = base + 2 * TILE_BYTES;   // stage: Q, dO
  uint8_t* s_ones = s_ring + STAGES * TILE_BYTES;
  uint8_t* s_stats = s_ones + AB_ONES;       // stage: logarithms, deltas
  __shared__ __align__(8) AbBars<CHAINS, STAGES> bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_found, s_shift;
  __shared__ AtPiece s_piece;

  const int tid = threadIdx.x, warp = warp_uniform(tid >> 5), lane = tid & 31;
  const int kv_heads = a.heads / a.group, rank = blockIdx.x % a.split, block = blockIdx.x / a.split;
  const int head = block % kv_heads, index = block / kv_heads;
  if (warp == 0) {
    AtPiece piece = {0, 0, 0, 0, 0};
    const bool found = at_find(a, AT_TILE, index, true, piece);
    if (lane == 0) {
      s_piece = piece;
      s_found = found;
    }
  }
  if (warp == LOADER && lane < 4) tma_prefetch_map(lane == 0 ? &a.q : lane == 1 ? &a.g : lane == 2 ? &a.k : &a.v);
  if (tid == 32) {
    bars.init(1, 2);
    s_abort = 0;
  }
  if (warp == ISSUER) tmem_alloc(&s_tmem, COLUMNS);
  // three ones to a row, zeros, and room for three parts of each statistic, zeros
  for (int i = tid; i < (AB_ONES + STAGES * AB_STATS) / 16; i += ab_threads(CHAINS))
    reinterpret_cast<uint4*>(s_ones)[i] = i < AT_TILE ? make_uint4(0x3F803F80u, 0x3F80u, 0, 0) : make_uint4(0, 0, 0, 0);
  psgd_fence_async_shared();
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  if (rank == 0) {
    at_clear_outside<T>(a, s_piece, (T*)a.dk, kv_heads, head, index);
    at_clear_outside<T>(a, s_piece, (T*)a.dv, kv_heads, head, index);
  }
  if (!s_found) {   // (so for all blocks of the cluster)
    psgd_wait_for_predecessor();
    if (warp == ISSUER) tmem_free(s_tmem, COLUMNS);
    return;
  }
  const uint32_t tmem = warp_uniform(s_tmem);
  const AtWait wait = {&s_abort, a.status};
  const int start = s_piece.start, length = warp_uniform(s_piece.length), k0 = warp_uniform(s_piece.piece) * AT_TILE;
  const int first = a.causal ? k0 / AT_STEP : 0;                      // first step of queries
  const int per_head = (length + AT_STEP - 1) / AT_STEP - first, heads = a.group / a.split, steps = per_head * heads;
  const int head0 = head * a.group + rank * heads;
  // Head and first query of a step, counted on without a division.
  struct Step {
    int head, row;
  };
  auto next = [&](Step& at, int by) {
    at.row += by * AT_STEP;
    while (at.row >= (first + per_head) * AT_STEP) {
      at.row -= per_head * AT_STEP;
      ++at.head;
    }
  };

  if (warp == LOADER) {
    {
      if (lane == 0) psgd_mbar_expect_tx(&bars.fixed, 2 * TILE_BYTES);
      if (lane == 0) {
        at_load_tile<PANELS, AT_TILE>(psgd_smem_u32(s_k), &a.k, head, start + k0, &bars.fixed);
        at_load_tile<PANELS, AT_TILE>(psgd_smem_u32(s_v), &a.v, head, start + k0, &bars.fixed);
      }
      Step step = {head0, first * AT_STEP}, later = step;
      const float per_log = -1.f / a.scale2;
      float x[4];      // of queries `lane` and `lane` + 32 of a step: minus the logarithm of the sum, as the products are scaled, and minus delta
      auto statistics = [&](const Step& at) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool in = at.row + lane + 32 * h < length;
          const long long from = (long long)at.head * a.tokens + start + at.row + lane + 32 * h;
          x[2 * h] = in ? a.lse[from] * per_log : 0.f;
          x[2 * h + 1] = in ? -a.delta[from] : 0.f;
        }
      };
      for (int i = 0; i < steps; ++i, next(step, 1)) {
        const int slot = i % STAGES;
        if (!wait(&bars.empty[slot], ((i / STAGES) & 1) ^ 1)) break;
        if (lane == 0) {
          psgd_mbar_expect_tx(&bars.full[slot], 2 * HALF);
          const uint32_t at = psgd_smem_u32(s_ring + slot * TILE_BYTES);
          at_load_tile<PANELS, AT_STEP>(at, &a.q, step.head, start + step.row, &bars.full[slot]);
          at_load_tile<PANELS, AT_STEP>(at + HALF, &a.g, step.head, start + step.row, &bars.full[slot]);
        }
        if (i == 0) {
          psgd_wait_for_predecessor();   // delta is complete
          statistics(step);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float high = __bfloat162float(__float2bfloat16_rn(x[e])), low = x[e] - high, middle = __bfloat162float(__float2bfloat16_rn(low));
          *reinterpret_cast<uint4*>(s_stats + slot * AB_STATS + (e & 1) * (AB_STATS / 2) + (lane + 32 * (e >> 1)) * 16) =
              make_uint4(pack2<__nv_bfloat16>(high, middle), pack2<__nv_bfloat16>(low - middle, 0.f), 0, 0);
        }
        psgd_fence_async_shared();
        __syncwarp();
        if (lane == 0) psgd_mbar_arrive(&bars.full[slot]);
        next(later, 1);
        if (i + 1 < steps) statistics(later);
      }
    }
    psgd_wait_for_predecessor();   // (nobody behind this grid may begin before the one before it has ended)
  } else if (warp == ISSUER) {
    const int k_steps = (a.size + 15) / 16;
    constexpr uint32_t S_SHAPE = umma_shape(AtType<T>::value, false, AT_STEP);
    const uint32_t o_shape = umma_shape(AtType<T>::value, true, k_steps * 16);
    const uint32_t k_at = warp_uniform(psgd_smem_u32(s_k)), v_at = k_at + TILE_BYTES, ring_at = k_at + 2 * TILE_BYTES;
    const uint32_t ones_at = ring_at + STAGES * TILE_BYTES, stats_at = ones_at + AB_ONES;
    constexpr uint32_t ONE_SHAPE = umma_shape(AtType<__nv_bfloat16>::value, false, AT_STEP);
    bool ok = wait(&bars.fixed, 0);
    int have = -1;
    Step step = {head0, first * AT_STEP};     // the one behind `have`
    auto there = [&](int i) {
      if (i > have) {
        ok = ok && wait(&bars.full[i % STAGES], (i / STAGES) & 1);
        have = i;
        const int queries = length - step.row;
        next(step, 1);
        if (ok && queries < AT_STEP) {
          at_clear_rows<PANELS, AT_STEP>(s_ring + i % STAGES * TILE_BYTES, queries);
          at_clear_rows<PANELS, AT_STEP>(s_ring + i % STAGES * TILE_BYTES + HALF, queries);
        }
      }
      if (ok) umma_fence_after();
      return ok;
    };
    auto scores = [&](int i) {
      if (!there(i)) return;
      umma_rows_by_rows<4 * PANELS, AT_STEP>(tmem + i % CHAINS * 128, k_at, ring_at + i % STAGES * TILE_BYTES, S_SHAPE, k_steps);
      umma_add_columns<AT_TILE, AT_STEP>(tmem + i % CHAINS * 128, ones_at, stats_at + i % STAGES * AB_STATS, ONE_SHAPE);
      umma_arrive(&bars.s[i % CHAINS]);
    };
    auto slopes = [&](int i) {
      if (!there(i)) return;
      umma_rows_by_rows<4 * PANELS, AT_STEP>(tmem + i % CHAINS * 128 + AT_STEP, v_at, ring_at + i % STAGES * TILE_BYTES + HALF, S_SHAPE, k_steps);
      umma_add_columns<AT_TILE, AT_STEP>(tmem + i % CHAINS * 128 + AT_STEP, ones_at, stats_at + i % STAGES * AB_STATS + AB_STATS / 2, ONE_SHAPE);
      umma_arrive(&bars.dp[i % CHAINS]);
    };
    for (int i = 0; i < CHAINS && i < steps && ok; ++i) {
      scores(i);
      if (ok) slopes(i);
    }
    for (int i = 0; i < steps && ok; ++i) {
      const int chain = i % CHAINS;
      const uint32_t parity = (i / CHAINS) & 1, stage = ring_at + i % STAGES * TILE_BYTES;
      ok = wait(&bars.p[chain], parity);
      if (!ok) break;
      umma_fence_after();
      umma_weights_by_rows<0, 4, AT_STEP, AB_GAP>(tmem + DV, tmem + chain * 128, stage + HALF, o_shape, i > 0);
      if (i + CHAINS < steps) scores(i + CHAINS);
      ok = ok && wait(&bars.ds[chain], parity);
      if (!ok) break;
      umma_fence_after();
      umma_weights_by_rows<0, 4, AT_STEP, AB_GAP>(tmem + DK, tmem + chain * 128 + AT_STEP, stage, o_shape, i > 0);
      if (length <= AB_FINE) umma_weights_by_rows<0, 4, AT_STEP, AB_GAP>(tmem + DK, tmem + chain * 128 + AT_STEP + AB_GAP, stage, o_shape, true);
      umma_arrive(&bars.empty[i % STAGES]);
      if (i + CHAINS < steps) slopes(i + CHAINS);
      if (i == steps - 1) umma_arrive(&bars.done);
    }
  } else {
    const int chain = warp >> 3, half = (warp >> 2) & 1, row = tid & 127, key = k0 + row;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = tmem + lanes + chain * 128 + half * AB_WIDE, dp_at = s_at + AT_STEP;
    Step step = {head0, first * AT_STEP};
    next(step, chain);
    bool ok = true;
    int mine = 0;                   // steps of this chain so far
    if (AB_SHIFTS<T>) {
      if (warp == 0) {              // (beside the warp that loads, which waits for the statistics)
        psgd_wait_for_predecessor();
        const int room = ab_room(a, head, start, length, true, first * AT_STEP / AT_TILE);
        if (lane == 0) s_shift = min(room, AB_MOST_SHIFT);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(256 * CHAINS) : "memory");
    }
    const int shift = AB_SHIFTS<T> ? s_shift : 0, lift = AB_SHIFTS<T> ? ab_lift(shift, length) : 0;     // of dS, of P
    for (int i = chain; i < steps; i += CHAINS, ++mine, next(step, CHAINS)) {
      const int q0 = step.row + half * AB_WIDE;      // this thread's first query
      ok = wait(&bars.s[chain], mine & 1);
      if (!ok) break;
      umma_fence_after();
      float p[AB_WIDE];
      tmem_load32(s_at, p);
      tmem_load_wait<AB_WIDE>(p);
#pragma unroll
      for (int c = 0; c < AB_WIDE; c += 2) {
        const float2 x = make_float2(p[c], p[c + 1]), factor = make_float2(a.scale2, a.scale2);
        const float2 y = AB_SHIFTS<T> ? fma2(x, factor, make_float2((float)lift, (float)lift)) : mul2(x, factor);
        p[c] = at_exp2(y.x);
        p[c + 1] = at_exp2(y.y);
      }
      if (a.causal && q0 < k0 + AT_TILE) {     // some queries come before some keys
        const int from = key - q0;
#pragma unroll
        for (int c = 0; c < AB_WIDE; ++c)
          if (c < from) p[c] = 0.f;
      }
      // (Queries behind the sequence have rows of zeros and deltas of zero: their weights are multiplied by zeros, their slopes are zeros.)
      uint32_t w[16];
#pragma unroll
      for (int e = 0; e < AB_WIDE; e += 2) w[e / 2] = pack2<T>(p[e], p[e + 1]);
      if (AB_SHIFTS<T> && shift < lift) {
        const float less = ab_power(shift - lift);
#pragma unroll
        for (int e = 0; e < AB_WIDE; ++e) p[e] *= less;
      }
      tmem_store16(s_at, w);
      tmem_store_wait();
      at_arrive(&bars.p[chain]);
      ok = wait(&bars.dp[chain], mine & 1);
      if (!ok) break;
      umma_fence_after();
      float d[AB_WIDE];
      tmem_load32(dp_at, d);
      tmem_load_wait<AB_WIDE>(d);
#pragma unroll
      for (int e = 0; e < AB_WIDE; e += 2) {
        const float2 f = mul2(make_float2(p[e], p[e + 1]), make_float2(d[e], d[e + 1]));
        w[e / 2] = pack2<T>(f.x, f.y);
        d[e] = f.x;
        d[e + 1] = f.y;
      }
      tmem_store16(dp_at, w);
      if (length <= AB_FINE) ab_store_rest<T>(dp_at + AB_GAP, d, w);
      tmem_store_wait();
      at_arrive(&bars.ds[chain]);
    }
    if (ok) ok = wait(&bars.done, 0);
    if (ok) {
      umma_fence_after();
      // dV and dK by four warps each; heads of more than 64 by the eight of a chain
      const int which = CHAINS == 2 ? chain : half, panel = CHAINS == 2 ? half : 0;
      const uint32_t at = tmem + lanes + (which == 0 ? DV : DK) + panel * 64;
      if (a.split == 1) {
        const int first_row = k0 + (warp & 3) * 32;
        at_write_rows<T, 1>(at, which == 0 ? 1.f / ab_power(lift) : a.scale / ab_power(shift), (which == 0 ? s_v : s_k) + (panel * 4 + (warp & 3)) * 4096,
                            (T*)(which == 0 ? a.dv : a.dk) + ((long long)(start + first_row) * kv_heads + head) * a.size + panel * 64, (T*)nullptr,
                            (long long)kv_heads * a.size, length - first_row, a.size - panel * 64);
      } else {
        // this block's share: [dV, dK][128 rows][64 PANELS] float32, groups of four elements where no two lanes meet in a bank
        float* share = reinterpret_cast<float*>(base) + (which * AT_TILE + row) * 64 * PANELS;
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          float f[32];
          tmem_load32(at + c, f);
          tmem_load_wait<32>(f);
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(share + ((panel * 64 + c + e) ^ ((row & 7) << 2))) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
        }
      }
    }
  }
  umma_fence_before();
  __syncthreads();
  if (s_abort) {
    psgd_let_copies_land();
    __syncthreads();
  }
  if (warp == ISSUER) {
    __syncwarp();
    tmem_free(tmem, COLUMNS);
  }
  if (a.split > 1) {
    // Rows rank, rank + split, ... of both, by this block. (Where a wait has run out somewhere the sums are not valid, and the
    // status word says so.)
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    constexpr int FOURS = 16 * PANELS;
    for (int e = tid; e < 2 * AT_TILE * FOURS; e += ab_threads(CHAINS)) {
      const int which = e / (AT_TILE * FOURS), r = e / FOURS % AT_TILE, c = e % FOURS * 4;
      if (r % a.split != rank || k0 + r >= length || c >= a.size) continue;
      float* at = reinterpret_cast<float*>(base) + (which * AT_TILE + r) * 64 * PANELS + (c ^ ((r & 7) << 2));
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int b = 0; b < a.split; ++b) {
        const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(at, b));
        sum.x += x.x;
        sum.y += x.y;
        sum.z += x.z;
        sum.w += x.w;
      }
      const int shift = AB_SHIFTS<T> ? s_shift : 0;      // (the same in all blocks)
      const float f = which == 0 ? 1.f / ab_power(AB_SHIFTS<T> ? ab_lift(shift, length) : 0) : a.scale / ab_power(shift);
      T* out = (T*)(which == 0 ? a.dv : a.dk) + ((long long)(start + k0 + r) * kv_heads + head) * a.size + c;
      *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(sum.x * f, sum.y * f), pack2<T>(sum.z * f, sum.w * f));
    }
    cluster.sync();   // nobody leaves while its share is read
  }
}

// ---- host --------------------------------------------------------------------------------------
typedef CUresult (*AtEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Tiles of queries per block of the forward pass.
constexpr int at_tiles(int size) { return size <= 64 ? 1 : 2; }

// [tokens, heads, size] with `row` and `head` elements between rows and heads: boxes of 64 elements of one head in 64 rows, zeros outside.
int at_encode(CUtensorMap* map, const void* at, int type, int tokens, int heads, int size, long long row, long long head) {
  static AtEncodeFn fn = nullptr;
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = (AtEncodeFn)p;
  }
  if (fn == nullptr) {
    psgd_set_error("cuTensorMapEncodeTiled is not available from this driver");
    return -1;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)size, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)head * 2, (cuuint64_t)row * 2};
  const cuuint32_t box[3] = {64, 1, 64}, elem[3] = {1, 1, 1};
  const CUresult rc = fn(map, type == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void*)at, dims, strides, box, elem,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) {
    psgd_set_error("cuTensorMapEncodeTiled failed with CUresult %d for [%d, %d, %d], strides %lld and %lld", (int)rc, tokens, heads, size, row, head);
    return -1;
  }
  return 0;
}

// Pieces of `rows` that the tokens of one head can make: each sequence may leave one unfilled.
long long at_most_pieces(int sequences, int tokens, int rows) { return (long long)tokens / rows + (sequences < tokens ? sequences : tokens); }

int at_fill(AtArgs& a, const void* q, const void* k, const void* v, const long long* strides, const int* offsets, int sequences, int tokens, int heads,
            int kv_heads, int size, int type, int causal, float scale, int rows, int grid_heads, int* status) {
  if (sequences < 1 || tokens < 1 || kv_heads < 1 || heads % kv_heads != 0 || size < 8 || size > 128 || size % 8 != 0) {
    psgd_set_error("packed attention: %d sequences, %d tokens, %d and %d heads of %d", sequences, tokens, heads, kv_heads, size);
    return -1;
  }
  // Encoding a tensor map is a call of the driver, which wants a context: a thread that has made no call of the runtime yet
  // (one of the autograd engine's) has none.
  int device = 0;
  PSGD_CUDA_OK(cudaGetDevice(&device));
  PSGD_CUDA_OK(cudaSetDevice(device));
  memset(&a, 0, sizeof(a));
  if (at_encode(&a.q, q, type, tokens, heads, size, strides[0], strides[1]) || at_encode(&a.k, k, type, tokens, kv_heads, size, strides[2], strides[3]) ||
      at_encode(&a.v, v, type, tokens, kv_heads, size, strides[4], strides[5]))
    return -1;
  a.offsets = offsets;
  a.sequences = sequences;
  a.tokens = tokens;
  a.heads = heads;
  a.group = heads / kv_heads;
  a.size = size;
  a.causal = causal;
  a.scale = scale;
  a.scale2 = scale * AT_LOG2E;
  const long long blocks = at_most_pieces(sequences, tokens, rows);
  if (blocks * grid_heads > 0x7fffffffll) {
    psgd_set_error("packed attention: %lld tiles of %d heads are more than a grid holds", blocks, grid_heads);
    return -1;
  }
  a.blocks = (int)blocks;
  a.status = status;
  return 0;
}

// Writes the order down where a warp cannot find it by itself. `plan`: psgd_attention_plan_ints of memory.
int at_plan(AtArgs& a, int rows, int* plan, cudaStream_t stream) {
  if (a.sequences <= 32) return 0;
  if (plan == nullptr) {
    psgd_set_error("packed attention: %d sequences need a plan", a.sequences);
    return -1;
  }
  a.plan = plan;
  return psgd_launch(psgd_attention_plan_kernel, a.tokens / rows + 1, AT_PLAN_THREADS, 0, stream, 0, a.offsets, a.sequences, a.tokens, rows, a.blocks, plan);
}

template <typename T, int PANELS>
int at_forward(const AtArgs& a, cudaStream_t stream) {
  constexpr int TILES = at_tiles(PANELS * 64);
  static unsigned long long devices = 0;
  if (const int code = psgd_allow_shared((const void*)psgd_attention_kernel<T, PANELS, TILES>, af_shared(PANELS, TILES), devices)) return code;
  return psgd_launch(psgd_attention_kernel<T, PANELS, TILES>, a.blocks * a.heads, af_threads(TILES), af_shared(PANELS, TILES), stream, 0, a);
}
template <typename T, int PANELS>
int at_backward(AtArgs a, cudaStream_t stream) {
  static unsigned long long q_devices = 0, kv_devices = 0;
  // A block of the keys' pass holds its tensor memory while it waits for the queries' pass to end, whose blocks may have begun without theirs: as many as
  // fit beside one of them must leave it enough.
  constexpr size_t SM_SHARED = 228 * 1024, OF_Q = ab_shared(PANELS, 0), OF_KV = ab_shared(PANELS, AB_ONES + ab_stages(PANELS) * AB_STATS);
  static_assert(((SM_SHARED - OF_Q) / OF_KV + 1) * 256 * PANELS <= 512, "tensor memory");
  if (const int code = psgd_allow_shared((const void*)psgd_attention_dq_kernel<T, PANELS>, ab_shared(PANELS, 0), q_devices)) return code;
  if (const int code = psgd_allow_shared((const void*)psgd_attention_dkv_kernel<T, PANELS>, ab_shared(PANELS, AB_ONES + ab_stages(PANELS) * AB_STATS), kv_devices)) return code;
  if constexpr (AB_SHIFTS<T>) {
    if (const int code = psgd_launch(psgd_attention_lengths_kernel, a.blocks * (a.heads / a.group), AN_THREADS, 0, stream, 0, a)) return code;
  }
  // (delta comes from the first)
  if (const int code = psgd_launch(psgd_attention_dq_kernel<T, PANELS>, a.blocks * a.heads, ab_threads(PANELS), ab_shared(PANELS, 0), stream, AB_SHIFTS<T>, a)) return code;
  const int kv_heads = a.heads / a.group;
  a.split = 1;
  for (int split = 2; split <= AB_MOST_SPLIT && split <= a.group && (long long)a.blocks * kv_heads * a.split < AB_ENOUGH; ++split)
    if (a.group % split == 0) a.split = split;
  if ((long long)a.blocks * kv_heads * a.split > 0x7fffffffll) a.split = 1;
  return psgd_launch_clusters(psgd_attention_dkv_kernel<T, PANELS>, a.blocks * kv_heads * a.split, ab_threads(PANELS), ab_shared(PANELS, AB_ONES + ab_stages(PANELS) * AB_STATS), stream, 1,
                              a.split, a);
}

}  // namespace

// Ints of scratch that a call needs as `plan`; with 0 it may be null.
PSGD_API long long psgd_attention_plan_ints(int sequences, int tokens) { return sequences <= 32 ? 0 : 1 + 3 * at_most_pieces(sequences, tokens, AT_TILE); }

// dtype: 1 bfloat16, 2 float16. strides: rows and heads of q, k and v, in elements, multiples of 8; addresses on 16-byte boundaries. `out` is
// [tokens, heads, size], contiguous, `rest` (what rounding takes from it: the backward pass wants it) likewise or null, lse [heads, tokens]. Rows of `out` outside the sequences become zeros.
PSGD_API int psgd_attention(const void* q, const void* k, const void* v, const long long* strides, const int* offsets, int sequences, int tokens, int heads,
                            int kv_heads, int size, int dtype, int causal, float scale, void* out, void* rest, float* lse, int* plan, int* status,
                            cudaStream_t stream) {
  AtArgs a;
  if (at_fill(a, q, k, v, strides, offsets, sequences, tokens, heads, kv_heads, size, dtype, causal, scale, at_tiles(size) * AT_TILE, heads, status)) return -1;
  a.out = out;
  a.rest = rest;
  a.lse = lse;
  if (const int code = at_plan(a, at_tiles(size) * AT_TILE, plan, stream)) return code;
  if (dtype == 1) return size <= 64 ? at_forward<__nv_bfloat16, 1>(a, stream) : at_forward<__nv_bfloat16, 2>(a, stream);
  return size <= 64 ? at_forward<__half, 1>(a, stream) : at_forward<__half, 2>(a, stream);
}

// strides: those of q, k, v and of the output's gradient. delta: scratch, [heads, tokens] words, float16 [2 heads + key heads, tokens]. dq, dk, dv are contiguous.
PSGD_API int psgd_attention_backward(const void* q, const void* k, const void* v, const void* grad, const long long* strides, const int* offsets, int sequences,
                                     int tokens, int heads, int kv_heads, int size, int dtype, int causal, float scale, const void* out, const void* rest, const float* lse,
                                     float* delta, void* dq, void* dk, void* dv, int* plan, int* status, cudaStream_t stream) {
  AtArgs a;
  if (at_fill(a, q, k, v, strides, offsets, sequences, tokens, heads, kv_heads, size, dtype, causal, scale, AT_TILE, heads, status)) return -1;
  if (at_encode(&a.g, grad, dtype, tokens, heads, size, strides[6], strides[7])) return -1;
  a.out = out;
  a.rest = rest;
  a.grad = grad;
  a.grad_row = strides[6];
  a.grad_head = strides[7];
  a.lse = (float*)lse;
  a.delta = delta;
  if (dtype != 1) {
    a.lengths_g = (int*)(delta + (long long)heads * tokens);
    a.lengths_v = a.lengths_g + (long long)heads * tokens;
  }
  a.value = v;
  a.value_row = strides[4];
  a.value_head = strides[5];
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  if (const int code = at_plan(a, AT_TILE, plan, stream)) return code;
  if (dtype == 1) return size <= 64 ? at_backward<__nv_bfloat16, 1>(a, stream) : at_backward<__nv_bfloat16, 2>(a, stream);
  return size <= 64 ? at_backward<__half, 1>(a, stream) : at_backward<__half, 2>(a, stream);
}
