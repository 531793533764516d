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
// All three kernels work on tiles of 128 x 128 scores. Rows of Q, K, V and dO come by TMA in tiles of 128 rows, and the
// scores never leave tensor memory and registers: a thread owns a row of a tile (a lane of tensor memory), so that a row's
// maximum and sum need no exchange between lanes, and P and dS go back to tensor memory as the A operand of the second products.
//   forward   a block has two tiles of queries of one head that share K and V. While the tensor core multiplies for one of
//             them, the four warps of the other take exponentials.
//   dQ        a block has one tile of queries and walks over keys.
//   dK, dV    a block has one tile of keys and walks over the queries of all heads of its group, transposed: lanes are
//             keys, so that P^T and dS^T are A operands as they come. Nothing is added with atomics: the same inputs
//             give the same bits. The price is that S and dP are computed twice (seven products instead of five).
// A row of a tile that belongs to another sequence, or lies behind the last one, may hold anything: scores with it are
// replaced, and where it would be multiplied by their zeros its row in shared memory is cleared.
//
// Blocks are dealt out with the longest first: the device finds the n-th tile in the order of its distance from the
// sequence's beginning (causal: of its work), from the offsets alone.
//
// Every wait is bounded: where one runs out, the block sets the status word, all its warps fall through, and the
// kernel ends.
#include <cuda.h>
#include <string.h>

#include "psgd_umma.cuh"

namespace {

constexpr int AT_TILE = 128;
constexpr float AT_LOG2E = 1.44269504088896341f;

struct AtArgs {
  CUtensorMap q, k, v, g;        // boxes of 64 elements x 1 head x 128 rows; g: the gradient of the output
  const int* offsets;
  int sequences, tokens, heads, group, size;   // group: query heads per key head
  int causal;
  float scale, scale2;           // scale, scale log2(e)
  int blocks;                    // tiles (forward: pairs of them) that the grid has room for, per head
  const void* out;               // forward: written; backward: read. [tokens, heads, size]
  const void* grad;              // the gradient of the output, as `g` addresses it
  long long grad_row, grad_head; // its strides
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

// ---- which tile --------------------------------------------------------------------------------
// Sequences cut into pieces of `rows`; piece number `index` in the order: the pieces that have the most of their sequence before them
// (`from_end`: behind them) first. One warp asks. Returns false where there are fewer.
struct AtPiece {
  int start, length, piece;      // first row and rows of its sequence, its number there
};
__device__ __forceinline__ int at_bound(const int* offsets, int s, int tokens) { return min(max(offsets[s], 0), tokens); }
__device__ bool at_find(const AtArgs& a, int rows, int index, bool from_end, AtPiece& out) {
  const int lane = threadIdx.x & 31;
  auto pieces = [&](int s) {
    if (s >= a.sequences) return 0;
    const int lo = at_bound(a.offsets, s, a.tokens), hi = at_bound(a.offsets, s + 1, a.tokens);
    return hi > lo ? (hi - lo + rows - 1) / rows : 0;
  };
  const int mine = pieces(lane);
  // pieces at level `level` of their sequences or above
  auto above = [&](int level) {
    int n = max(mine - level, 0);
    for (int s = lane + 32; s < a.sequences; s += 32) n += max(pieces(s) - level, 0);
    return (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
  };
  int most = mine;
  for (int s = lane + 32; s < a.sequences; s += 32) most = max(most, pieces(s));
  most = (int)__reduce_max_sync(0xffffffffu, (unsigned)most);
  if (index >= above(0)) return false;
  int lo = 0, hi = most;         // above(lo) > index >= above(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (above(mid) > index) lo = mid;
    else hi = mid;
  }
  int left = index - above(lo + 1);   // the left-th sequence with more than `lo` pieces
  for (int s0 = 0; s0 < a.sequences; s0 += 32) {
    const bool has = (s0 ? pieces(s0 + lane) : mine) > lo;
    const unsigned votes = __ballot_sync(0xffffffffu, has);
    const int n = __popc(votes);
    if (left >= n) {
      left -= n;
      continue;
    }
    const int s = s0 + __fns(votes, 0, left + 1);
    out.start = at_bound(a.offsets, s, a.tokens);
    out.length = at_bound(a.offsets, s + 1, a.tokens) - out.start;
    out.piece = from_end ? (out.length + rows - 1) / rows - 1 - lo : lo;
    return true;
  }
  return false;
}

// Rows of a result that belong to no sequence: zeros. Dealt out over the blocks of a head.
template <typename T>
__device__ void at_clear_outside(const AtArgs& a, T* out, int heads, int head, int block) {
  const int first = at_bound(a.offsets, 0, a.tokens), last = at_bound(a.offsets, a.sequences, a.tokens);
  const int outside = first + a.tokens - max(first, last);
  for (int i = block; i < outside; i += a.blocks) {
    const int row = i < first ? i : max(first, last) + i - first;
    T* p = out + ((long long)row * heads + head) * a.size;
    for (int e = threadIdx.x; e < a.size; e += blockDim.x) p[e] = T(0.f);
  }
}

// ---- pieces of the pipelines -------------------------------------------------------------------
struct AtWait {
  volatile int* abort_flag;
  int* status;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
#pragma unroll 1
    for (int i = 0; i < 16; ++i)   // (the clock is read only when it takes longer)
      if (psgd_mbar_try_wait(bar, parity)) return true;
    return psgd_mbar_wait(bar, parity, abort_flag, status);
  }
};

// A tile of 128 rows from `row` of one head: PANELS boxes of 64 elements.
template <int PANELS>
__device__ __forceinline__ void at_load_tile(uint32_t dst, const CUtensorMap* map, int head, int row, uint64_t* bar) {
#pragma unroll
  for (int p = 0; p < PANELS; ++p) tma_load_box3(dst + p * UMMA_PANEL, map, p * 64, head, row, bar);
}

// Clears rows [from, 128) of a tile, by threads that have one row each.
template <int PANELS>
__device__ __forceinline__ void at_clear_row(uint8_t* tile, int row, int from) {
  if (row < from) return;
#pragma unroll
  for (int p = 0; p < PANELS; ++p) {
    uint4* at = reinterpret_cast<uint4*>(tile + p * UMMA_PANEL + row * 128);
#pragma unroll
    for (int i = 0; i < 8; ++i) at[i] = make_uint4(0, 0, 0, 0);
  }
}

// `columns` of an accumulator's row, times `factor`, as a row of 16-bit numbers.
template <typename T, int PANELS>
__device__ __forceinline__ void at_write_row(uint32_t tmem, float factor, T* row, int size, bool write) {
#pragma unroll
  for (int c = 0; c < PANELS * 64; c += 32) {
    if (c >= size) break;
    float f[32];
    tmem_load32(tmem + c, f);
    tmem_load_wait();
    if (write) {
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        if (c + i < size)
          *reinterpret_cast<uint4*>(row + c + i) = make_uint4(pack2<T>(f[i] * factor, f[i + 1] * factor), pack2<T>(f[i + 2] * factor, f[i + 3] * factor),
                                                              pack2<T>(f[i + 4] * factor, f[i + 5] * factor), pack2<T>(f[i + 6] * factor, f[i + 7] * factor));
      }
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
constexpr int AF_THREADS = 320;   // warps 0-3 and 4-7: one tile of queries each; 8: loads; 9: products
constexpr int AF_RING = 4;        // tiles of K and V under way

template <int PANELS>
constexpr size_t af_shared() { return 1024 + (size_t)(2 + AF_RING) * PANELS * UMMA_PANEL; }

template <typename T, int PANELS>
__global__ void __launch_bounds__(AF_THREADS, 1) psgd_attention_kernel(const __grid_constant__ AtArgs a) {
  constexpr int TILE_BYTES = PANELS * UMMA_PANEL;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = base;
  uint8_t* s_ring = base + 2 * TILE_BYTES;
  __shared__ __align__(8) uint64_t bar_q, bar_full[AF_RING], bar_empty[AF_RING], bar_s[2], bar_p[2], bar_o[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_found;
  __shared__ AtPiece s_piece;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.x % a.heads, index = blockIdx.x / a.heads;
  at_clear_outside<T>(a, (T*)a.out, a.heads, head, index);
  if (warp == 0) {
    AtPiece piece = {0, 0, 0};
    const bool found = at_find(a, 2 * AT_TILE, index, false, piece);
    if (lane == 0) {
      s_piece = piece;
      s_found = found;
    }
  }
  if (tid == 32) {
    psgd_mbar_init(&bar_q, 1);
    for (int i = 0; i < AF_RING; ++i) {
      psgd_mbar_init(&bar_full[i], 1);
      psgd_mbar_init(&bar_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      psgd_mbar_init(&bar_s[t], 1);
      psgd_mbar_init(&bar_p[t], 128);
      psgd_mbar_init(&bar_o[t], 1);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (!s_found) return;
  if (warp == 9) tmem_alloc(&s_tmem, 512);
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  const uint32_t tmem = s_tmem;
  const AtWait wait = {&s_abort, a.status};
  const int start = s_piece.start, length = s_piece.length, row0 = s_piece.piece * 2 * AT_TILE;
  // tiles of keys that each tile of queries meets
  int n[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int q0 = row0 + t * AT_TILE;
    n[t] = q0 >= length ? 0 : a.causal ? q0 / AT_TILE + 1 : (length + AT_TILE - 1) / AT_TILE;
  }
  const int steps = max(n[0], n[1]);

  if (warp == 8) {
    if (lane == 0) {
      psgd_mbar_expect_tx(&bar_q, n[1] > 0 ? 2 * TILE_BYTES : TILE_BYTES);
      for (int t = 0; t < 2; ++t)
        if (n[t] > 0) at_load_tile<PANELS>(psgd_smem_u32(s_q + t * TILE_BYTES), &a.q, head, start + row0 + t * AT_TILE, &bar_q);
      for (int i = 0; i < 2 * steps; ++i) {   // K_0, V_0, K_1, V_1, ...
        const int slot = i % AF_RING;
        if (!wait(&bar_empty[slot], ((i / AF_RING) & 1) ^ 1)) break;
        psgd_mbar_expect_tx(&bar_full[slot], TILE_BYTES);
        at_load_tile<PANELS>(psgd_smem_u32(s_ring + slot * TILE_BYTES), (i & 1) ? &a.v : &a.k, head / a.group, start + (i >> 1) * AT_TILE, &bar_full[slot]);
      }
    }
  } else if (warp == 9) {
    if (lane == 0) {
      const int k_steps = (a.size + 15) / 16;
      constexpr uint32_t S_SHAPE = umma_shape(AtType<T>::value, false, AT_TILE);
      const uint32_t o_shape = umma_shape(AtType<T>::value, true, k_steps * 16);
      const uint32_t q_at = psgd_smem_u32(s_q), ring_at = psgd_smem_u32(s_ring);
      auto scores = [&](int t, int j) {
        umma_rows_by_rows(tmem + t * AT_TILE, q_at + t * TILE_BYTES, ring_at + (2 * j % AF_RING) * TILE_BYTES, S_SHAPE, k_steps, false);
        umma_arrive(&bar_s[t]);
      };
      bool ok = wait(&bar_q, 0) && wait(&bar_full[0], 0);
      if (ok) {
        umma_fence_after();
        for (int t = 0; t < 2; ++t)
          if (n[t] > 0) scores(t, 0);
        umma_arrive(&bar_empty[0]);
      }
      for (int j = 0; j < steps && ok; ++j) {
        const int kv = 2 * j + 1, kn = 2 * j + 2;
        ok = wait(&bar_full[kv % AF_RING], (kv / AF_RING) & 1);
        bool next = false;
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= n[t]) continue;
          ok = wait(&bar_p[t], j & 1);
          if (!ok) break;
          umma_fence_after();
          for (int s = 0; s < AT_TILE / 16; ++s)
            umma_ts(tmem + 2 * AT_TILE + t * AT_TILE, tmem + t * AT_TILE + s * 8, umma_tile(ring_at + (kv % AF_RING) * TILE_BYTES + s * 2048), o_shape, j > 0 || s > 0);
          umma_arrive(&bar_o[t]);
          if (j + 1 < n[t]) {
            if (!next) ok = wait(&bar_full[kn % AF_RING], (kn / AF_RING) & 1);
            if (!ok) break;
            next = true;
            umma_fence_after();
            scores(t, j + 1);
          }
        }
        if (!ok) break;
        umma_arrive(&bar_empty[kv % AF_RING]);
        if (j + 1 < steps) umma_arrive(&bar_empty[kn % AF_RING]);
      }
    }
  } else {
    const int t = warp >> 2, row = tid & 127;
    const int q = row0 + t * AT_TILE + row;          // in its sequence
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * AT_TILE, o_at = tmem + lanes + 2 * AT_TILE + t * AT_TILE;
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
      tmem_load_wait();
      if (j == n[t] - 1) {
        const int last = limit - j * AT_TILE;
#pragma unroll
        for (int c = 0; c < AT_TILE; ++c)
          if (c > last) s[c] = -INFINITY;
        const int held = length - j * AT_TILE;       // keys of this tile that belong to the sequence
        if (held < AT_TILE) {
          const int kv = 2 * j + 1;
          ok = wait(&bar_full[kv % AF_RING], (kv / AF_RING) & 1);
          if (!ok) break;
          at_clear_row<PANELS>(s_ring + (kv % AF_RING) * TILE_BYTES, row, held);
          psgd_fence_async_shared();
        }
      }
      float most[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < AT_TILE; ++c) most[c & 3] = fmaxf(most[c & 3], s[c]);
      const float largest = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
      // The sums stay relative to an older maximum while exponents stay below 2^8: accumulators are rescaled only when it moves by more.
      const bool moves = (largest - m) * a.scale2 > 8.f || j == 0;
      if (j > 0) {
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
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= f;
            tmem_store16(o_at + c, reinterpret_cast<uint32_t*>(o));
            tmem_store16(o_at + c + 16, reinterpret_cast<uint32_t*>(o) + 16);
          }
        }
      } else {
        m = largest;
      }
      const float from = m == -INFINITY ? 0.f : m * a.scale2;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < AT_TILE; c += 32) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float x = at_exp2(fmaf(s[c + i], a.scale2, -from)), y = at_exp2(fmaf(s[c + i + 1], a.scale2, -from));
          sum[i & 3] += x;
          sum[(i & 3) + 1] += y;
          p[i / 2] = pack2<T>(x, y);
        }
        tmem_store16(s_at + c / 2, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_store_wait();
      umma_fence_before();
      psgd_mbar_arrive(&bar_p[t]);
    }
    if (ok && n[t] > 0) ok = wait(&bar_o[t], (n[t] - 1) & 1);
    if (ok && n[t] > 0) {
      umma_fence_after();
      const bool held = q < length;
      T* out = (T*)a.out + ((long long)(start + (held ? q : 0)) * a.heads + head) * a.size;
      at_write_row<T, PANELS>(o_at, 1.f / l, out, a.size, held);
      if (held) a.lse[(long long)head * a.tokens + start + q] = m * a.scale2 + log2f(l);
    }
  }
  umma_fence_before();
  __syncthreads();
  if (s_abort) {
    psgd_let_copies_land();
    __syncthreads();
  }
  if (warp == 9) {
    __syncwarp();
    tmem_free(tmem, 512);
  }
}

// ---- backward ----------------------------------------------------------------------------------
constexpr int AB_THREADS = 320;   // warps 0-7: scores (0-3 columns 0-63 of a tile, 4-7 the others); 8: loads; 9: products

template <int PANELS>
constexpr size_t ab_shared() { return 1024 + (size_t)6 * PANELS * UMMA_PANEL; }   // two tiles that stay, two stages of two that pass

struct AbBars {
  uint64_t fixed, full[2], empty[2], s, dp, p, ds, done;
};

__device__ __forceinline__ void ab_init(AbBars& b) {
  psgd_mbar_init(&b.fixed, 1);
  for (int i = 0; i < 2; ++i) {
    psgd_mbar_init(&b.full[i], 1);
    psgd_mbar_init(&b.empty[i], 1);
  }
  psgd_mbar_init(&b.s, 1);
  psgd_mbar_init(&b.dp, 1);
  psgd_mbar_init(&b.p, 256);
  psgd_mbar_init(&b.ds, 256);
  psgd_mbar_init(&b.done, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

// dQ: tensor memory holds S (128 columns), dP (128; dS takes its place in halves of 32 columns at 0 and 64) and dQ.
// S of the next tile is multiplied as soon as this one is in registers, dP of the next behind dQ of this one.
template <typename T, int PANELS>
__global__ void __launch_bounds__(AB_THREADS, 1) psgd_attention_dq_kernel(const __grid_constant__ AtArgs a) {
  constexpr int TILE_BYTES = PANELS * UMMA_PANEL;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = base;
  uint8_t* s_g = base + TILE_BYTES;
  uint8_t* s_ring = base + 2 * TILE_BYTES;   // stage: K, V
  __shared__ __align__(8) AbBars bars;
  __shared__ float s_delta[AT_TILE];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_found;
  __shared__ AtPiece s_piece;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.x % a.heads, index = blockIdx.x / a.heads;
  at_clear_outside<T>(a, (T*)a.dq, a.heads, head, index);
  if (warp == 0) {
    AtPiece piece = {0, 0, 0};
    const bool found = at_find(a, AT_TILE, index, false, piece);
    if (lane == 0) {
      s_piece = piece;
      s_found = found;
    }
  }
  if (tid == 32) {
    ab_init(bars);
    s_abort = 0;
  }
  __syncthreads();
  if (!s_found) return;
  if (warp == 9) tmem_alloc(&s_tmem, 512);
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  const uint32_t tmem = s_tmem;
  const AtWait wait = {&s_abort, a.status};
  const int start = s_piece.start, length = s_piece.length, q0 = s_piece.piece * AT_TILE;
  const int steps = a.causal ? s_piece.piece + 1 : (length + AT_TILE - 1) / AT_TILE;
  constexpr int DP = AT_TILE, DQ = 2 * AT_TILE;   // columns

  if (warp == 8) {
    if (lane == 0) {
      psgd_mbar_expect_tx(&bars.fixed, 2 * TILE_BYTES);
      at_load_tile<PANELS>(psgd_smem_u32(s_q), &a.q, head, start + q0, &bars.fixed);
      at_load_tile<PANELS>(psgd_smem_u32(s_g), &a.g, head, start + q0, &bars.fixed);
      for (int j = 0; j < steps; ++j) {
        const int slot = j & 1;
        if (!wait(&bars.empty[slot], ((j >> 1) & 1) ^ 1)) break;
        psgd_mbar_expect_tx(&bars.full[slot], 2 * TILE_BYTES);
        const uint32_t at = psgd_smem_u32(s_ring + slot * 2 * TILE_BYTES);
        at_load_tile<PANELS>(at, &a.k, head / a.group, start + j * AT_TILE, &bars.full[slot]);
        at_load_tile<PANELS>(at + TILE_BYTES, &a.v, head / a.group, start + j * AT_TILE, &bars.full[slot]);
      }
    }
  } else if (warp == 9) {
    if (lane == 0) {
      const int k_steps = (a.size + 15) / 16;
      constexpr uint32_t S_SHAPE = umma_shape(AtType<T>::value, false, AT_TILE);
      const uint32_t q_shape = umma_shape(AtType<T>::value, true, k_steps * 16);
      const uint32_t q_at = psgd_smem_u32(s_q), g_at = psgd_smem_u32(s_g), ring_at = psgd_smem_u32(s_ring);
      auto scores = [&](int j) {
        umma_rows_by_rows(tmem, q_at, ring_at + (j & 1) * 2 * TILE_BYTES, S_SHAPE, k_steps, false);
        umma_arrive(&bars.s);
      };
      auto slopes = [&](int j) {
        umma_rows_by_rows(tmem + DP, g_at, ring_at + (j & 1) * 2 * TILE_BYTES + TILE_BYTES, S_SHAPE, k_steps, false);
        umma_arrive(&bars.dp);
      };
      bool ok = wait(&bars.fixed, 0) && wait(&bars.full[0], 0);
      if (ok) {
        umma_fence_after();
        scores(0);
        slopes(0);
      }
      for (int j = 0; j < steps && ok; ++j) {
        ok = wait(&bars.p, j & 1);    // S is in registers
        if (!ok) break;
        umma_fence_after();
        if (j + 1 < steps) {
          ok = wait(&bars.full[(j + 1) & 1], ((j + 1) >> 1) & 1);
          if (!ok) break;
          umma_fence_after();
          scores(j + 1);
        }
        ok = wait(&bars.ds, j & 1);
        if (!ok) break;
        umma_fence_after();
        for (int s = 0; s < AT_TILE / 16; ++s)
          umma_ts(tmem + DQ, tmem + DP + (s >> 2) * 64 + (s & 3) * 8, umma_tile(ring_at + (j & 1) * 2 * TILE_BYTES + s * 2048), q_shape, j > 0 || s > 0);
        umma_arrive(&bars.empty[j & 1]);
        if (j + 1 < steps) slopes(j + 1);
        else umma_arrive(&bars.done);
      }
    }
  } else {
    const int half = warp >> 2, row = tid & 127, q = q0 + row;
    const bool held = q < length;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const long long stat = (long long)head * a.tokens + start + q;
    // delta of the row, once for the keys' pass too
    if (half == 0) {
      float d = 0.f;
      if (held) {
        const T* o = (const T*)a.out + ((long long)(start + q) * a.heads + head) * a.size;
        const T* g = (const T*)a.grad + (long long)(start + q) * a.grad_row + (long long)head * a.grad_head;
        for (int c = 0; c < a.size; c += 8) {
          const uint4 x = *reinterpret_cast<const uint4*>(o + c), y = *reinterpret_cast<const uint4*>(g + c);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 u = unpack2<T>(xs[i]), v = unpack2<T>(ys[i]);
            d = fmaf(u.x, v.x, d);
            d = fmaf(u.y, v.y, d);
          }
        }
        a.delta[stat] = d;
      }
      s_delta[row] = d;
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const float delta = s_delta[row], lse = held ? a.lse[stat] : 0.f;
    const int limit = (a.causal ? min(q, length - 1) : length - 1) - half * 64;
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      ok = wait(&bars.s, j & 1);
      if (!ok) break;
      umma_fence_after();
      float p[64];
      tmem_load32(tmem + lanes + half * 64, p);
      tmem_load32(tmem + lanes + half * 64 + 32, p + 32);
      tmem_load_wait();
      umma_fence_before();
      psgd_mbar_arrive(&bars.p);
      const bool edge = j == steps - 1;
      const int last = limit - j * AT_TILE;
#pragma unroll
      for (int c = 0; c < 64; ++c) p[c] = at_exp2(fmaf(p[c], a.scale2, -lse));
      if (edge) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c > last) p[c] = 0.f;
        const int keys = length - j * AT_TILE;
        if (keys < AT_TILE) {
          ok = wait(&bars.full[j & 1], (j >> 1) & 1);
          if (!ok) break;
          if (half == 0) at_clear_row<PANELS>(s_ring + (j & 1) * 2 * TILE_BYTES, row, keys);
          psgd_fence_async_shared();
        }
      }
      ok = wait(&bars.dp, j & 1);
      if (!ok) break;
      umma_fence_after();
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        float d[32];
        tmem_load32(tmem + lanes + DP + half * 64 + c, d);
        tmem_load_wait();
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float x = p[c + i] * (d[i] - delta), y = p[c + i + 1] * (d[i + 1] - delta);
          if (edge) {   // (a masked key may hold anything)
            if (c + i > last) x = 0.f;
            if (c + i + 1 > last) y = 0.f;
          }
          w[i / 2] = pack2<T>(x, y);
        }
        tmem_store16(tmem + lanes + DP + half * 64 + c / 2, w);
      }
      tmem_store_wait();
      umma_fence_before();
      psgd_mbar_arrive(&bars.ds);
    }
    if (ok) ok = wait(&bars.done, 0);
    if (ok) {
      umma_fence_after();
      if (half == 0) {
        T* out = (T*)a.dq + ((long long)(start + (held ? q : 0)) * a.heads + head) * a.size;
        at_write_row<T, PANELS>(tmem + lanes + DQ, a.scale, out, a.size, held);
      }
    }
  }
  umma_fence_before();
  __syncthreads();
  if (s_abort) {
    psgd_let_copies_land();
    __syncthreads();
  }
  if (warp == 9) {
    __syncwarp();
    tmem_free(tmem, 512);
  }
}

// dK, dV: tensor memory holds S^T (P^T takes its place), dP^T (dS^T likewise), dV and dK: 4 x 128 columns. dV of a tile and S^T of the
// next are multiplied while dS^T is formed, dK and dP^T of the next while the next exponentials are taken.
template <typename T, int PANELS>
__global__ void __launch_bounds__(AB_THREADS, 1) psgd_attention_dkv_kernel(const __grid_constant__ AtArgs a) {
  constexpr int TILE_BYTES = PANELS * UMMA_PANEL;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* s_k = base;
  uint8_t* s_v = base + TILE_BYTES;
  uint8_t* s_ring = base + 2 * TILE_BYTES;   // stage: Q, dO
  __shared__ __align__(8) AbBars bars;
  __shared__ __align__(16) float s_lse[3][AT_TILE], s_delta[3][AT_TILE];   // of tile i in place i % 3, see below
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_found;
  __shared__ AtPiece s_piece;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kv_heads = a.heads / a.group, head = blockIdx.x % kv_heads, index = blockIdx.x / kv_heads;
  at_clear_outside<T>(a, (T*)a.dk, kv_heads, head, index);
  at_clear_outside<T>(a, (T*)a.dv, kv_heads, head, index);
  if (warp == 0) {
    AtPiece piece = {0, 0, 0};
    const bool found = at_find(a, AT_TILE, index, true, piece);
    if (lane == 0) {
      s_piece = piece;
      s_found = found;
    }
  }
  if (tid == 32) {
    ab_init(bars);
    s_abort = 0;
  }
  __syncthreads();
  if (!s_found) return;
  if (warp == 9) tmem_alloc(&s_tmem, 512);
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  const uint32_t tmem = s_tmem;
  const AtWait wait = {&s_abort, a.status};
  const int start = s_piece.start, length = s_piece.length, k0 = s_piece.piece * AT_TILE;
  const int first = a.causal ? s_piece.piece : 0;                     // first tile of queries
  const int per_head = (length + AT_TILE - 1) / AT_TILE - first, steps = per_head * a.group;
  constexpr int DP = AT_TILE, DV = 2 * AT_TILE, DK = 3 * AT_TILE;     // columns
  auto q_head = [&](int i) { return head * a.group + i / per_head; };
  auto q_row = [&](int i) { return (first + i % per_head) * AT_TILE; };

  if (warp == 8) {
    if (lane == 0) {
      psgd_mbar_expect_tx(&bars.fixed, 2 * TILE_BYTES);
      at_load_tile<PANELS>(psgd_smem_u32(s_k), &a.k, head, start + k0, &bars.fixed);
      at_load_tile<PANELS>(psgd_smem_u32(s_v), &a.v, head, start + k0, &bars.fixed);
      for (int i = 0; i < steps; ++i) {
        const int slot = i & 1;
        if (!wait(&bars.empty[slot], ((i >> 1) & 1) ^ 1)) break;
        psgd_mbar_expect_tx(&bars.full[slot], 2 * TILE_BYTES);
        const uint32_t at = psgd_smem_u32(s_ring + slot * 2 * TILE_BYTES);
        at_load_tile<PANELS>(at, &a.q, q_head(i), start + q_row(i), &bars.full[slot]);
        at_load_tile<PANELS>(at + TILE_BYTES, &a.g, q_head(i), start + q_row(i), &bars.full[slot]);
      }
    }
  } else if (warp == 9) {
    if (lane == 0) {
      const int k_steps = (a.size + 15) / 16;
      constexpr uint32_t S_SHAPE = umma_shape(AtType<T>::value, false, AT_TILE);
      const uint32_t o_shape = umma_shape(AtType<T>::value, true, k_steps * 16);
      const uint32_t k_at = psgd_smem_u32(s_k), v_at = psgd_smem_u32(s_v), ring_at = psgd_smem_u32(s_ring);
      auto scores = [&](int i) {
        umma_rows_by_rows(tmem, k_at, ring_at + (i & 1) * 2 * TILE_BYTES, S_SHAPE, k_steps, false);
        umma_arrive(&bars.s);
      };
      auto slopes = [&](int i) {
        umma_rows_by_rows(tmem + DP, v_at, ring_at + (i & 1) * 2 * TILE_BYTES + TILE_BYTES, S_SHAPE, k_steps, false);
        umma_arrive(&bars.dp);
      };
      // the halves of P^T and dS^T lie 64 columns apart
      auto second = [&](uint32_t d, uint32_t p, uint32_t tile, bool more) {
        for (int s = 0; s < AT_TILE / 16; ++s) umma_ts(tmem + d, tmem + p + (s >> 2) * 64 + (s & 3) * 8, umma_tile(tile + s * 2048), o_shape, more || s > 0);
      };
      bool ok = wait(&bars.fixed, 0) && wait(&bars.full[0], 0);
      if (ok) {
        umma_fence_after();
        scores(0);
        slopes(0);
      }
      for (int i = 0; i < steps && ok; ++i) {
        const uint32_t stage = ring_at + (i & 1) * 2 * TILE_BYTES;
        ok = wait(&bars.p, i & 1);
        if (!ok) break;
        umma_fence_after();
        second(DV, 0, stage + TILE_BYTES, i > 0);
        if (i + 1 < steps) {
          ok = wait(&bars.full[(i + 1) & 1], ((i + 1) >> 1) & 1);
          if (!ok) break;
          umma_fence_after();
          scores(i + 1);
        }
        ok = wait(&bars.ds, i & 1);
        if (!ok) break;
        umma_fence_after();
        second(DK, DP, stage, i > 0);
        umma_arrive(&bars.empty[i & 1]);
        if (i + 1 < steps) slopes(i + 1);
        else umma_arrive(&bars.done);
      }
    }
  } else {
    const int half = warp >> 2, row = tid & 127, key = k0 + row;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    auto statistic = [&](int i) {   // of query `row` of tile i: log of the sum, or delta
      const int q = q_row(i) + row;
      if (q >= length) return 0.f;
      return (half == 0 ? a.lse : a.delta)[(long long)q_head(i) * a.tokens + start + q];
    };
    float (*mine)[AT_TILE] = half == 0 ? s_lse : s_delta;
    mine[0][row] = statistic(0);
    asm volatile("bar.sync 1, 256;" ::: "memory");
    bool ok = true;
    for (int i = 0; i < steps; ++i) {
      const float ahead = i + 1 < steps ? statistic(i + 1) : 0.f;
      const int q0 = q_row(i) + half * 64, queries = length - q_row(i);
      // queries [from, to) of this thread's columns meet its key
      const int from = a.causal ? key - q0 : 0, to = length - q0;
      const bool edge = (a.causal && i % per_head == 0) || queries < AT_TILE;
      // The statistics of tile i were written before the arrivals for tile i - 1. A warp may be behind by the second half of a tile, no
      // more: two places would not do, three do.
      ok = (i == 0 || wait(&bars.p, (i - 1) & 1)) && wait(&bars.s, i & 1);
      if (!ok) break;
      umma_fence_after();
      float p[64];
      tmem_load32(tmem + lanes + half * 64, p);
      tmem_load32(tmem + lanes + half * 64 + 32, p + 32);
      tmem_load_wait();
      const float4* lse = reinterpret_cast<const float4*>(&s_lse[i % 3][half * 64]);
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const float4 x = lse[c / 4];
        p[c] = at_exp2(fmaf(p[c], a.scale2, -x.x));
        p[c + 1] = at_exp2(fmaf(p[c + 1], a.scale2, -x.y));
        p[c + 2] = at_exp2(fmaf(p[c + 2], a.scale2, -x.z));
        p[c + 3] = at_exp2(fmaf(p[c + 3], a.scale2, -x.w));
      }
      if (edge) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (c < from || c >= to) p[c] = 0.f;
        if (queries < AT_TILE) {
          ok = wait(&bars.full[i & 1], (i >> 1) & 1);
          if (!ok) break;
          at_clear_row<PANELS>(s_ring + (i & 1) * 2 * TILE_BYTES + half * TILE_BYTES, row, queries);
          psgd_fence_async_shared();
        }
      }
      // S^T is 128 columns wide and P^T takes 32 of each half: a half is written by the warps that read it
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) w[e / 2] = pack2<T>(p[c + e], p[c + e + 1]);
        tmem_store16(tmem + lanes + half * 64 + c / 2, w);
      }
      mine[(i + 1) % 3][row] = ahead;
      tmem_store_wait();
      umma_fence_before();
      psgd_mbar_arrive(&bars.p);
      ok = wait(&bars.dp, i & 1);
      if (!ok) break;
      umma_fence_after();
      const float4* delta = reinterpret_cast<const float4*>(&s_delta[i % 3][half * 64]);
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        float d[32];
        tmem_load32(tmem + lanes + DP + half * 64 + c, d);
        tmem_load_wait();
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 x = delta[(c + e) / 4];
          float f[4] = {p[c + e] * (d[e] - x.x), p[c + e + 1] * (d[e + 1] - x.y), p[c + e + 2] * (d[e + 2] - x.z), p[c + e + 3] * (d[e + 3] - x.w)};
          if (edge) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (c + e + u < from || c + e + u >= to) f[u] = 0.f;
          }
          w[e / 2] = pack2<T>(f[0], f[1]);
          w[e / 2 + 1] = pack2<T>(f[2], f[3]);
        }
        tmem_store16(tmem + lanes + DP + half * 64 + c / 2, w);
      }
      tmem_store_wait();
      umma_fence_before();
      psgd_mbar_arrive(&bars.ds);
    }
    if (ok) ok = wait(&bars.done, 0);
    if (ok) {
      umma_fence_after();
      const bool held = key < length;
      T* out = (T*)(half == 0 ? a.dv : a.dk) + ((long long)(start + (held ? key : 0)) * kv_heads + head) * a.size;
      at_write_row<T, PANELS>(tmem + lanes + (half == 0 ? DV : DK), half == 0 ? 1.f : a.scale, out, a.size, held);
    }
  }
  umma_fence_before();
  __syncthreads();
  if (s_abort) {
    psgd_let_copies_land();
    __syncthreads();
  }
  if (warp == 9) {
    __syncwarp();
    tmem_free(tmem, 512);
  }
}

// ---- host --------------------------------------------------------------------------------------
typedef CUresult (*AtEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// [tokens, heads, size] with `row` and `head` elements between rows and heads: boxes of 64 elements of one head in 128 rows, zeros outside.
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
  const cuuint32_t box[3] = {64, 1, AT_TILE}, elem[3] = {1, 1, 1};
  const CUresult rc = fn(map, type == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void*)at, dims, strides, box, elem,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) {
    psgd_set_error("cuTensorMapEncodeTiled failed with CUresult %d for [%d, %d, %d], strides %lld and %lld", (int)rc, tokens, heads, size, row, head);
    return -1;
  }
  return 0;
}

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
  const long long blocks = (long long)tokens / rows + (sequences < tokens ? sequences : tokens);   // each sequence may leave one piece unfilled
  if (blocks * grid_heads > 0x7fffffffll) {
    psgd_set_error("packed attention: %lld tiles of %d heads are more than a grid holds", blocks, grid_heads);
    return -1;
  }
  a.blocks = (int)blocks;
  a.status = status;
  return 0;
}

template <typename T, int PANELS>
int at_forward(const AtArgs& a, cudaStream_t stream) {
  static unsigned long long devices = 0;
  if (const int code = psgd_allow_shared((const void*)psgd_attention_kernel<T, PANELS>, af_shared<PANELS>(), devices)) return code;
  return psgd_launch(psgd_attention_kernel<T, PANELS>, a.blocks * a.heads, AF_THREADS, af_shared<PANELS>(), stream, 0, a);
}
template <typename T, int PANELS>
int at_backward(const AtArgs& a, cudaStream_t stream) {
  static unsigned long long q_devices = 0, kv_devices = 0;
  if (const int code = psgd_allow_shared((const void*)psgd_attention_dq_kernel<T, PANELS>, ab_shared<PANELS>(), q_devices)) return code;
  if (const int code = psgd_allow_shared((const void*)psgd_attention_dkv_kernel<T, PANELS>, ab_shared<PANELS>(), kv_devices)) return code;
  // (delta comes from the first)
  if (const int code = psgd_launch(psgd_attention_dq_kernel<T, PANELS>, a.blocks * a.heads, AB_THREADS, ab_shared<PANELS>(), stream, 0, a)) return code;
  return psgd_launch(psgd_attention_dkv_kernel<T, PANELS>, a.blocks * (a.heads / a.group), AB_THREADS, ab_shared<PANELS>(), stream, 0, a);
}

}  // namespace

// dtype: 1 bfloat16, 2 float16. strides: rows and heads of q, k and v, in elements, multiples of 8; addresses on 16-byte boundaries. `out` is
// [tokens, heads, size], contiguous, lse [heads, tokens]. Rows of `out` outside the sequences become zeros.
PSGD_API int psgd_attention(const void* q, const void* k, const void* v, const long long* strides, const int* offsets, int sequences, int tokens, int heads,
                            int kv_heads, int size, int dtype, int causal, float scale, void* out, float* lse, int* status, cudaStream_t stream) {
  AtArgs a;
  if (at_fill(a, q, k, v, strides, offsets, sequences, tokens, heads, kv_heads, size, dtype, causal, scale, 2 * AT_TILE, heads, status)) return -1;
  a.out = out;
  a.lse = lse;
  if (dtype == 1) return size <= 64 ? at_forward<__nv_bfloat16, 1>(a, stream) : at_forward<__nv_bfloat16, 2>(a, stream);
  return size <= 64 ? at_forward<__half, 1>(a, stream) : at_forward<__half, 2>(a, stream);
}

// strides: those of q, k, v and of the output's gradient. delta: scratch, [heads, tokens]. dq, dk, dv are contiguous.
PSGD_API int psgd_attention_backward(const void* q, const void* k, const void* v, const void* grad, const long long* strides, const int* offsets, int sequences,
                                     int tokens, int heads, int kv_heads, int size, int dtype, int causal, float scale, const void* out, const float* lse,
                                     float* delta, void* dq, void* dk, void* dv, int* status, cudaStream_t stream) {
  AtArgs a;
  if (at_fill(a, q, k, v, strides, offsets, sequences, tokens, heads, kv_heads, size, dtype, causal, scale, AT_TILE, heads, status)) return -1;
  if (at_encode(&a.g, grad, dtype, tokens, heads, size, strides[6], strides[7])) return -1;
  a.out = out;
  a.grad = grad;
  a.grad_row = strides[6];
  a.grad_head = strides[7];
  a.lse = (float*)lse;
  a.delta = delta;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  if (dtype == 1) return size <= 64 ? at_backward<__nv_bfloat16, 1>(a, stream) : at_backward<__nv_bfloat16, 2>(a, stream);
  return size <= 64 ? at_backward<__half, 1>(a, stream) : at_backward<__half, 2>(a, stream);
}
