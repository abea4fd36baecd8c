// Matrix product in 8-bit integers with a scale for each token and each
// output channel:
//   y[m, n] = (sum_k a[m, k] w[n, k]) * sa[m] * sw[n] + bias[n]
// a int8 [m, k] (rows8.cuh), w int8 [n, k].  tcgen05.mma kind::i8 sums exactly
// in int32 (k < 131072), whatever the split; the scaling is fp32, rounded once
// to the output's type.  K is walked in steps of 128 bytes (one 128-byte
// swizzle row); TMA fills what lies past K, M or N with zeros.
//
//  * gemm8_few_kernel: up to 16 tokens, without TMEM or TMA (see there).
//  * gemm8_tile_kernel: one tile of 128 channels x T tokens (T <= 256, a
//    multiple of 16) for each cluster of up to 8 CTAs, which split K between
//    them and add their sums through distributed shared memory.  Channels are
//    the MMA's M side, so that few tokens cost few columns.  Bound by its fixed
//    cost, about 5 us: 400 x 4,096 x 1,024 9 us, 1,600 x 1,024 x 8,192 15.8 us.
//  * gemm8_pair_kernel: persistent CTA pairs (cta_group::2), tiles of 256
//    tokens x 256 channels, the accumulators double buffered so that a tile's
//    epilogue runs under the next one's products.  Bound by the tensor pipe:
//    6,208 x 2,048 x 16,384 141 us (2.95 POP/s, 86 % of the pipe's cycles; 90 %
//    of twice the bf16 rate that a library product reaches).
#pragma once

#include "attention8.cuh"
#include "rows8.cuh"

namespace w4a4 {

struct alignas(64) Gemm8Params {
  CUtensorMap tmap_a;  // tokens: int8 {k, m}, box {128, T or 128}, SW128
  CUtensorMap tmap_w;  // weights: int8 {k, n}, box {128, 128}, SW128
  CUtensorMap tmap_y;  // output {n, m}, box {64 bytes, 32}, SW64 (pair kernel, tma_store)
  const float* sa;
  const float* sw;
  const void* bias;    // output type, or NULL
  void* y;             // contiguous [m, n]
  long long m;
  int n;
  int k_steps;         // ceil(k / 128)
  int tok_tile;        // T (tile kernel)
  int stages;
  int n_tok_tiles, n_w_tiles;
  int tma_store;       // rows of y begin at multiples of 16 bytes
  unsigned long long wait_limit_ns;
};

constexpr int kG8StepBytes = 128;             // K bytes of a step
constexpr int kG8ABytes = 128 * kG8StepBytes;  // 16 KB of weights (or tokens) of a step
constexpr int kG8MaxStages = 12;

// Scales and biases of four consecutive channels from n on (zero past N).
template <typename T>
struct G8Channels {
  float w[4], b[4];
  bool vec;  // the four exist, and rows of y keep vectors of four aligned
  __device__ __forceinline__ G8Channels(const Gemm8Params& p, int n) : vec(n + 4 <= p.n && p.n % 4 == 0) {
    const T* bias = static_cast<const T*>(p.bias);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = n + i < p.n ? __ldg(p.sw + n + i) : 0.f;
      b[i] = bias && n + i < p.n ? to_float(bias[n + i]) : 0.f;
    }
  }
  // sums of one token -> y
  __device__ __forceinline__ void store(const Gemm8Params& p, long long m, int n, const int4& acc, float sa) const {
    const float4 v = make_float4(fmaf(static_cast<float>(acc.x) * sa, w[0], b[0]), fmaf(static_cast<float>(acc.y) * sa, w[1], b[1]),
                                 fmaf(static_cast<float>(acc.z) * sa, w[2], b[2]), fmaf(static_cast<float>(acc.w) * sa, w[3], b[3]));
    T* dst = static_cast<T*>(p.y) + m * p.n + n;
    if (vec) {
      store4(dst, v);
    } else {
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.n) dst[i] = from_float<T>(x[i]);
    }
  }
};

// Shared memory: the ring of `stages` (16 KB of weights, T rows of tokens),
// which the sums [T][128] and what the other CTAs of the cluster send take
// over once the products are done; token scales; barriers.
constexpr int kG8TileThreads = 256;
constexpr int kG8TileMax = 256;  // tokens
__host__ __device__ constexpr int gemm8_tile_ring(int tok_tile, int stages, bool split) {
  const int ring = stages * (kG8ABytes + tok_tile * kG8StepBytes), sums = (split ? 2 : 1) * tok_tile * 512;
  return ring > sums ? ring : sums;
}
__host__ __device__ constexpr int gemm8_tile_smem(int tok_tile, int stages, bool split) {
  const int need = gemm8_tile_ring(tok_tile, stages, split) + kG8TileMax * 4 + (2 * kG8MaxStages + 2) * 8 + 16 + 1024;
  return need > kOneCtaSmem ? need : kOneCtaSmem;
}

// grid.x = cluster size x token tiles x weight tiles (token tiles fastest, so
// that the CTAs of one weight tile run side by side).
template <typename T>
__global__ void __launch_bounds__(kG8TileThreads) gemm8_tile_kernel(const __grid_constant__ Gemm8Params p) {
  extern __shared__ uint8_t g8_smem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(g8_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  const int S = p.stages, tok_bytes = p.tok_tile * kG8StepBytes;
  const int ranks = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
  uint8_t* w_ring = base;                    // [S][16 KB]
  uint8_t* t_ring = base + S * kG8ABytes;    // [S][T x 128]
  int* sums = reinterpret_cast<int*>(base);  // [T][128], after the products
  float* tok_scale = reinterpret_cast<float*>(base + gemm8_tile_ring(p.tok_tile, S, ranks > 1));  // [256]
  uint64_t* bars = reinterpret_cast<uint64_t*>(tok_scale + kG8TileMax);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kG8MaxStages + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const auto bar_full = [&](int s) { return smem_addr(bars + s); };
  const auto bar_empty = [&](int s) { return smem_addr(bars + kG8MaxStages + s); };
  const uint32_t bar_acc = smem_addr(bars + 2 * kG8MaxStages), bar_recv = smem_addr(bars + 2 * kG8MaxStages + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / ranks;
  const int wt = tile / p.n_tok_tiles, tt = tile - wt * p.n_tok_tiles;
  const int n0 = wt * 128;
  const long long m0 = static_cast<long long>(tt) * p.tok_tile;
  const int per = (p.k_steps + ranks - 1) / ranks;
  const int k0 = min(p.k_steps, rank * per), steps = min(p.k_steps, k0 + per) - k0;
  const uint32_t cols = p.tok_tile <= 32 ? 32 : p.tok_tile <= 64 ? 64 : p.tok_tile <= 128 ? 128 : 256;
  unsigned* err = &g_w4a4_device_error;
  const uint64_t limit = p.wait_limit_ns;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    mbar_init(bar_acc, 1);
    mbar_init(bar_recv, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_a);
    tma_prefetch_desc(&p.tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(smem_addr(tmem_slot), cols);
    tmem_relinquish();
  }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      RingPos st;
      int issued = 0;
      for (int i = 0; i < steps; ++i) {
        if (i >= S && !mbar_wait_bounded(bar_empty(st.idx), st.phase ^ 1u, abort_flag, err, kErrWaitEmpty, limit)) break;
        mbar_arrive_expect_tx(bar_full(st.idx), static_cast<uint32_t>(kG8ABytes + tok_bytes));
        tma_load_2d(smem_addr(w_ring + st.idx * kG8ABytes), &p.tmap_w, (k0 + i) * kG8StepBytes, n0, bar_full(st.idx));
        tma_load_2d(smem_addr(t_ring + st.idx * tok_bytes), &p.tmap_a, (k0 + i) * kG8StepBytes, static_cast<int>(m0),
                    bar_full(st.idx));
        st.advance(S);
        ++issued;
      }
      // no copy may be in flight when the ring becomes the sums' buffer
      for (int i = 0; i < S && i < issued; ++i) {
        const int last = i + ((issued - 1 - i) / S) * S;
        volatile int no_abort = 0;
        mbar_wait_bounded(bar_full(i), (last / S) & 1, &no_abort, err, kErrWaitDrain, limit);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool issuer = elect_one();
    const uint32_t idesc = idesc_i8(128, p.tok_tile);
    RingPos st;
    for (int i = 0; i < steps; ++i) {
      if (!warp_all(mbar_wait_fast(bar_full(st.idx), st.phase, abort_flag, err, kErrWaitTma, limit))) break;
      tc_fence_after();
      const uint64_t ad = smem_desc_sw128(smem_addr(w_ring + st.idx * kG8ABytes));
      const uint64_t bd = smem_desc_sw128(smem_addr(t_ring + st.idx * tok_bytes));
      if (issuer) {
        umma_i8_ss(tmem_base, ad, bd, idesc, i > 0);
        umma_i8_ss(tmem_base, ad + 2, bd + 2, idesc, 1u);
        umma_i8_ss(tmem_base, ad + 4, bd + 4, idesc, 1u);
        umma_i8_ss(tmem_base, ad + 6, bd + 6, idesc, 1u);
        umma_commit(bar_empty(st.idx));
      }
      __syncwarp();
      st.advance(S);
    }
    if (issuer) umma_commit(bar_acc);
    __syncwarp();
  }
  // scales for the results below, under the products
  const int quarter = warp & 3;
  const uint32_t tacc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
  if (threadIdx.x < p.tok_tile) tok_scale[threadIdx.x] = m0 + threadIdx.x < p.m ? __ldg(p.sa + m0 + threadIdx.x) : 0.f;
  volatile int no_abort = 0;
  if (ranks == 1) {
    // ---- straight from TMEM: thread = channel, a column = a token, so a warp
    // writes 32 consecutive channels of one token at a time
    const int n = n0 + quarter * 32 + lane;
    const float sw = n < p.n ? __ldg(p.sw + n) : 0.f;
    const float bias = p.bias && n < p.n ? to_float(static_cast<const T*>(p.bias)[n]) : 0.f;
    __syncthreads();  // tok_scale
    const bool good = mbar_wait_bounded(bar_acc, 0, &no_abort, err, kErrWaitAccum, limit) && !*abort_flag;
    tc_fence_after();
    const int rows = static_cast<int>(min(static_cast<long long>(p.tok_tile), p.m - m0));
    T* dst = static_cast<T*>(p.y) + m0 * p.n + n;
    for (int c0 = (warp >> 2) * 16; c0 < p.tok_tile; c0 += 64) {
      uint32_t r[2][16];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (c0 + 32 * i < p.tok_tile) tmem_ld_32x32b_x16(tacc + c0 + 32 * i, r[i]);
      tmem_ld_wait();
      if (!good || n >= p.n) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int t = c0 + 32 * i + j;
          if (t < rows)
            dst[static_cast<long long>(t) * p.n] =
                from_float<T>(fmaf(static_cast<float>(static_cast<int>(r[i][j])) * tok_scale[t], sw, bias));
        }
    }
    tc_fence_before();
    __syncthreads();
  } else {
    const G8Channels<T> channels(p, n0 + 4 * lane);  // a lane's four channels of the tile
    mbar_wait_bounded(bar_acc, 0, &no_abort, err, kErrWaitAccum, limit);
    tc_fence_after();
    __syncthreads();  // the producer has seen its copies land: the ring is free
    // ---- sums to shared memory: lane = channel, so a column's 128 are one line
    const int share = p.tok_tile / ranks;  // tokens that each CTA of the cluster finishes
    for (int c0 = (warp >> 2) * 16; c0 < p.tok_tile; c0 += 64) {
      uint32_t r[2][16];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (steps > 0 && c0 + 32 * i < p.tok_tile) {
          tmem_ld_32x32b_x16(tacc + c0 + 32 * i, r[i]);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) r[i][j] = 0u;
        }
      }
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (c0 + 32 * i < p.tok_tile)
#pragma unroll
          for (int j = 0; j < 16; ++j) sums[(c0 + 32 * i + j) * 128 + quarter * 32 + lane] = static_cast<int>(r[i][j]);
    }
    tc_fence_before();
    // ---- every CTA sends each other one its share of the sums, one bulk copy
    // each (loads from remote shared memory move a fraction of what these do)
    const int first = rank * share;
    int* recv = sums + p.tok_tile * 128;  // [ranks - 1][share][128]
    if (threadIdx.x == 0) mbar_arrive_expect_tx(bar_recv, static_cast<uint32_t>((ranks - 1) * share * 512));
    fence_proxy_async_smem();
    cluster_sync();  // sums written, barriers armed, rings free in all of them
    if (warp == 0 && lane < ranks && lane != rank)
      bulk_copy_s2cluster(mapa_shared(smem_addr(recv + (rank < lane ? rank : rank - 1) * share * 128), lane),
                          smem_addr(sums + lane * share * 128), static_cast<uint32_t>(share * 512),
                          mapa_shared(bar_recv, lane));
    __syncwarp();
    mbar_wait_bounded_cl(bar_recv, 0, &no_abort, err, kErrWaitAccum, limit);
    const bool aborted = *abort_flag != 0;
    const int4* own = reinterpret_cast<const int4*>(sums + first * 128) + lane;
    const int4* others = reinterpret_cast<const int4*>(recv) + lane;
#pragma unroll 2
    for (int t = warp; t < share; t += 8) {
      int4 acc = own[t * 32];
#pragma unroll
      for (int r = 0; r < 7; ++r) {
        if (r + 1 >= ranks) break;
        const int4 x = others[(r * share + t) * 32];
        acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
      }
      const long long m = m0 + first + t;
      if (!aborted && m < p.m && n0 + 4 * lane < p.n) channels.store(p, m, n0 + 4 * lane, acc, tok_scale[first + t]);
    }
    cluster_sync();  // no CTA leaves before its copies have been received
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, cols);
  }
}

// -------------------------------------------------------- few tokens (<= 16)
// One CTA of 8 or 16 warps per 8 NT channels; the warps share K in runs of 64 bytes
// and add their sums through shared memory.  mma.sync m16n8k32: the 16 rows are
// the tokens, the 8 columns weight rows; as K may be permuted when both
// operands agree, lane (g, t) loads 16 consecutive bytes of row g at 64 c + 16 t
// of both straight from global memory, two steps of MMA, with no set-up before
// the first weight is asked for.  Bound: the weights' way from HBM, and for a
// small product the launch and one trip to memory.  1 x 2,048 x 2,560 3.0 us, the
// tile kernel 5.1; 16 x 2,048 x 32,768 17.3 us (3.9 TB/s) and 20.4.
constexpr int kG8FewTokens = 16;

__device__ __forceinline__ void mma_s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Gemm8FewParams {
  const int8_t* a;
  const int8_t* w;
  const float* sa;
  const float* sw;
  const void* bias;
  void* y;
  long long lda, ldw;
  int m, n, k;
};

// 16 bytes of a row of k bytes at byte e, zeros past k (rows begin at multiples of 16 bytes and the
// last vector of a row that ends inside it is still within the row's stride).
__device__ __forceinline__ uint4 g8_load_tail(const int8_t* row, int e, int k) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (e < k) {
    v = __ldg(reinterpret_cast<const uint4*>(row + e));
    uint32_t* w = &v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int bytes = k - e - 4 * i;
      if (bytes <= 0) w[i] = 0u;
      else if (bytes < 4) w[i] &= (1u << (8 * bytes)) - 1u;
    }
  }
  return v;
}

template <typename T, bool HALF, int NT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) gemm8_few_kernel(const __grid_constant__ Gemm8FewParams p) {
  constexpr int R = HALF ? 8 : 16;
  __shared__ int part[WARPS][R][8 * NT];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 8 * NT;
  int acc[NT][4] = {};
  // rows that do not exist read the last one: their sums are not used
  const int8_t* a0 = p.a + min(g, p.m - 1) * p.lda + 16 * t;
  const int8_t* a1 = p.a + min(g + 8, p.m - 1) * p.lda + 16 * t;
  const int8_t* w[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) w[i] = p.w + static_cast<long long>(min(n0 + 8 * i + g, p.n - 1)) * p.ldw + 16 * t;
  const int full = p.k / 64;  // runs of 64 bytes: warp, warp + WARPS, ...
  const auto product = [&](const uint4& x0, const uint4& x1, const uint4 (&b)[NT]) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      mma_s8_16832(acc[i], x0.x, x1.x, x0.y, x1.y, b[i].x, b[i].y);
      mma_s8_16832(acc[i], x0.z, x1.z, x0.w, x1.w, b[i].z, b[i].w);
    }
  };
  constexpr int U = 4;  // runs whose loads are under way together
  int c = warp;
  for (; c + WARPS * (U - 1) < full; c += WARPS * U) {
    uint4 x0[U], x1[U], b[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = 64 * (c + WARPS * u);
#pragma unroll
      for (int i = 0; i < NT; ++i) b[u][i] = __ldg(reinterpret_cast<const uint4*>(w[i] + e));
      x0[u] = __ldg(reinterpret_cast<const uint4*>(a0 + e));
      x1[u] = HALF ? make_uint4(0u, 0u, 0u, 0u) : __ldg(reinterpret_cast<const uint4*>(a1 + e));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) product(x0[u], x1[u], b[u]);
  }
  for (; 64 * c < p.k; c += WARPS) {
    const int e = 64 * c;
    uint4 b[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) b[i] = g8_load_tail(w[i], e, p.k - 16 * t);
    const uint4 x0 = g8_load_tail(a0, e, p.k - 16 * t);
    const uint4 x1 = HALF ? make_uint4(0u, 0u, 0u, 0u) : g8_load_tail(a1, e, p.k - 16 * t);
    product(x0, x1, b);
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    *reinterpret_cast<int2*>(&part[warp][g][8 * i + 2 * t]) = make_int2(acc[i][0], acc[i][1]);
    if constexpr (!HALF) *reinterpret_cast<int2*>(&part[warp][g + 8][8 * i + 2 * t]) = make_int2(acc[i][2], acc[i][3]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * 8 * NT; i += 32 * WARPS) {
    const int r = i / (8 * NT), n = n0 + i % (8 * NT);
    if (r >= p.m || n >= p.n) continue;
    int sum = 0;
#pragma unroll
    for (int x = 0; x < WARPS; ++x) sum += part[x][r][i % (8 * NT)];
    const float b = p.bias ? to_float(static_cast<const T*>(p.bias)[n]) : 0.f;
    static_cast<T*>(p.y)[static_cast<long long>(r) * p.n + n] =
        from_float<T>(fmaf(static_cast<float>(sum) * __ldg(p.sa + r), __ldg(p.sw + n), b));
  }
}

// ---------------------------------------------------------------- CTA pairs
// Tiles of 256 tokens (128 in each CTA: the MMA's M side) x 256 channels (128
// weight rows in each CTA's shared memory).  Warp 0 loads, warp 1 of the
// leader issues, warps 2-9 are the epilogue: thread = token row, a warp takes
// 32 tokens x 128 channels in boxes of 64 bytes a row, which TMA stores carry
// off while the next box is converted.  The next tile's scales are loaded under
// this tile's epilogue.
constexpr int kG8PairStages = 5;
constexpr int kG8PairWarps = 10;
constexpr int kG8PairThreads = 32 * kG8PairWarps;
constexpr int kG8PairSmem = kG8PairStages * 2 * kG8ABytes + 8 * 4096 + 8 * 2 * 128 * 4 + (2 * kG8PairStages + 5) * 8 + 16 + 1024;

__device__ __forceinline__ void tma_store_2d(const void* tmap, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(src), "r"(x), "r"(y)
               : "memory");
}
// Waits until at most one committed bulk group of this thread has yet to read its source.
__device__ __forceinline__ void bulk_wait_group_read1() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }

template <typename T>
__global__ void __launch_bounds__(kG8PairThreads, 1) gemm8_pair_kernel(const __grid_constant__ Gemm8Params p) {
  extern __shared__ uint8_t g8_smem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(g8_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr int S = kG8PairStages;
  uint8_t* t_ring = base;                        // [S][128 tokens x 128]
  uint8_t* w_ring = base + S * kG8ABytes;        // [S][128 weight rows x 128]
  uint8_t* out_stage = base + 2 * S * kG8ABytes;  // [epilogue warp][2][32 rows][64 B], 64-byte swizzle
  float* chan = reinterpret_cast<float*>(out_stage + 8 * 4096);  // [epilogue warp][scale, bias][128 channels]
  uint64_t* bars = reinterpret_cast<uint64_t*>(chan + 8 * 2 * 128);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // full[s]   leader: both CTAs' halves of step i landed (every copy completes on the leader's barrier)
  // empty[s]  both (multicast commit): the products of step i are done
  // accfull / accempty[2]: accumulator hand-over (accempty lives in the leader)
  const auto bar_full = [&](int s) { return smem_addr(bars + s); };
  const auto bar_empty = [&](int s) { return smem_addr(bars + S + s); };
  const auto bar_accfull = [&](int b) { return smem_addr(bars + 2 * S + b); };
  const auto bar_accempty = [&](int b) { return smem_addr(bars + 2 * S + 2 + b); };
  const uint32_t bar_drain = smem_addr(bars + 2 * S + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int total = p.n_tok_tiles * p.n_w_tiles;
  unsigned* err = &g_w4a4_device_error;
  const uint64_t limit = p.wait_limit_ns;
  // token tiles fastest: the pairs that run together share few weight tiles
  const auto tile_m = [&](int t) { return static_cast<long long>(t % p.n_tok_tiles) * 256 + rank * 128; };
  const auto tile_n = [&](int t) { return (t / p.n_tok_tiles) * 256; };

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_accfull(b), 1);
      mbar_init(bar_accempty(b), 16);  // the epilogue warps of both CTAs
    }
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_a);
    tma_prefetch_desc(&p.tmap_w);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_addr(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  pdl_wait();
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------ TMA producer (lane 0, both CTAs)
    if (lane == 0) {
      RingPos st;
      int issued = 0;
      bool alive = true;
      for (int tile = pair; alive && tile < total; tile += n_pairs) {
        const int m0 = static_cast<int>(tile_m(tile)), n0 = tile_n(tile) + static_cast<int>(rank) * 128;
        for (int kt = 0; kt < p.k_steps; ++kt) {
          if (issued >= S &&
              !mbar_wait_bounded_cl(bar_empty(st.idx), st.phase ^ 1u, abort_flag, err, kErrWaitEmpty, limit)) {
            alive = false;
            break;
          }
          const uint32_t full = bar_full(st.idx);
          if (leader) mbar_arrive_expect_tx(full, 4 * kG8ABytes);
          tma_load_2d_pair(smem_addr(t_ring + st.idx * kG8ABytes), &p.tmap_a, kt * kG8StepBytes, m0, full);
          tma_load_2d_pair(smem_addr(w_ring + st.idx * kG8ABytes), &p.tmap_w, kt * kG8StepBytes, n0, full);
          st.advance(S);
          ++issued;
        }
      }
      // both CTAs' copies complete on the leader's barriers; the exit cluster barrier keeps the peer until then
      if (leader)
        for (int i = 0; i < S && i < issued; ++i) {
          const int last = i + ((issued - 1 - i) / S) * S;
          volatile int no_abort = 0;
          mbar_wait_bounded_cl(bar_full(i), (last / S) & 1, &no_abort, err, kErrWaitDrain, limit);
        }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (leader, whole warp; one lane issues)
    if (leader) {
      const bool issuer = elect_one();
      const uint64_t adesc = smem_desc_sw128(smem_addr(t_ring)), bdesc = smem_desc_sw128(smem_addr(w_ring));
      const uint32_t idesc = idesc_i8(256, 256);
      RingPos st;
      int count = 0;
      bool alive = true;
      for (int tile = pair; alive && tile < total; tile += n_pairs, ++count) {
        const int buf = count & 1;
        if (count >= 2 &&
            !warp_all(mbar_wait_bounded_cl(bar_accempty(buf), ((count >> 1) - 1) & 1, abort_flag, err, kErrWaitAccum, limit)))
          break;
        tc_fence_after();
        const uint32_t d = tmem_base + buf * 256;
        for (int kt = 0; kt < p.k_steps; ++kt) {
          const uint32_t full = bar_full(st.idx);
          if (!warp_all(mbar_try_wait_cl(full, st.phase) ||
                        mbar_wait_bounded_cl(full, st.phase, abort_flag, err, kErrWaitTma, limit))) {
            alive = false;
            break;
          }
          tc_fence_after();
          const uint64_t ad = adesc + static_cast<uint64_t>(st.idx * kG8ABytes >> 4);
          const uint64_t bd = bdesc + static_cast<uint64_t>(st.idx * kG8ABytes >> 4);
          if (issuer) {
            umma_i8_ss_pair(d, ad, bd, idesc, kt != 0);
            umma_i8_ss_pair(d, ad + 2, bd + 2, idesc, 1u);
            umma_i8_ss_pair(d, ad + 4, bd + 4, idesc, 1u);
            umma_i8_ss_pair(d, ad + 6, bd + 6, idesc, 1u);
            umma_commit_pair_mc(bar_empty(st.idx), 0x3);
          }
          __syncwarp();
          st.advance(S);
        }
        if (alive && issuer) umma_commit_pair_mc(bar_accfull(buf), 0x3);
        __syncwarp();
      }
      if (issuer) umma_commit_pair_mc(bar_drain, 0x3);
      __syncwarp();
    }
    if (lane == 0) {
      volatile int no_abort = 0;
      mbar_wait_bounded_cl(bar_drain, 0, &no_abort, err, kErrWaitDrain, limit);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ epilogue (warps 2-9, both CTAs)
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    float* sc = chan + (warp - 2) * 256;
    uint8_t* stage = out_stage + (warp - 2) * 4096;
    constexpr int W = 64 / sizeof(T);   // columns of a box: 32, or 16 of fp32
    constexpr int V = 16 / sizeof(T);   // of a 16-byte chunk
    constexpr int NC = 128 / W;
    // scales and biases of a tile: lane's four channels (32 apart) and its token
    float cs[4], cb[4], sa = 0.f;
    const auto load_scales = [&](int tile) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = tile_n(tile) + half * 128 + 32 * j + lane;
        cs[j] = n < p.n ? __ldg(p.sw + n) : 0.f;
        cb[j] = p.bias && n < p.n ? to_float(static_cast<const T*>(p.bias)[n]) : 0.f;
      }
      const long long m = tile_m(tile) + quarter * 32 + lane;
      sa = m < p.m ? __ldg(p.sa + m) : 0.f;
    };
    if (pair < total) load_scales(pair);
    int count = 0;
    for (int tile = pair; tile < total; tile += n_pairs, ++count) {
      const int buf = count & 1, n0 = tile_n(tile) + half * 128;  // the warp's 128 channels
      const long long m0 = tile_m(tile) + quarter * 32;           // and 32 tokens
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sc[32 * j + lane] = cs[j];
        sc[128 + 32 * j + lane] = cb[j];
      }
      const float sat = sa;
      __syncwarp();
      if (tile + n_pairs < total) load_scales(tile + n_pairs);
      if (!warp_all(mbar_wait_bounded_cl(bar_accfull(buf), (count >> 1) & 1, abort_flag, err, kErrWaitAccum, limit))) break;
      tc_fence_after();
      const uint32_t acc = tmem_base + lane_addr + buf * 256 + half * 128;
      uint32_t r[2][W];
      const auto load_acc = [&](int i) {
#pragma unroll
        for (int c = 0; c < W; c += 16)
          tmem_ld_32x32b_x16(acc + i * W + c, *reinterpret_cast<uint32_t(*)[16]>(&r[i & 1][c]));
      };
      load_acc(0);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        tmem_ld_wait();
        if (i + 1 < NC) {
          load_acc(i + 1);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(mapa_shared(bar_accempty(buf), 0));
        }
        uint8_t* box = stage + (i & 1) * 2048;
        bulk_wait_group_read1();  // (lane 0) the store of the box before last has read it
        __syncwarp();
#pragma unroll
        for (int x = 0; x < W; x += V) {
          float v[V];
#pragma unroll
          for (int y = 0; y < V; y += 4) {
            const float4 w = *reinterpret_cast<const float4*>(sc + i * W + x + y);
            const float4 b = *reinterpret_cast<const float4*>(sc + 128 + i * W + x + y);
            const uint32_t* q = &r[i & 1][x + y];
            v[y] = fmaf(static_cast<float>(static_cast<int>(q[0])) * sat, w.x, b.x);
            v[y + 1] = fmaf(static_cast<float>(static_cast<int>(q[1])) * sat, w.y, b.y);
            v[y + 2] = fmaf(static_cast<float>(static_cast<int>(q[2])) * sat, w.z, b.z);
            v[y + 3] = fmaf(static_cast<float>(static_cast<int>(q[3])) * sat, w.w, b.w);
          }
          T* dst = reinterpret_cast<T*>(box + lane * 64 + (((x / V) ^ ((lane >> 1) & 3)) << 4));
          if constexpr (V == 8) store8(dst, v);
          else *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        }
        const int n = n0 + i * W;
        if (p.tma_store) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (n < p.n && m0 < p.m) tma_store_2d(&p.tmap_y, smem_addr(box), n, static_cast<int>(m0));
            bulk_commit_group();
          }
        } else {
          // rows that do not begin at multiples of 16 bytes: 8, 4 or 2 bytes a lane
          __syncwarp();
          const auto by = [&](auto word) {
            using X = decltype(word);
            constexpr int E = sizeof(X) / sizeof(T);       // values of a lane
            constexpr int L = 64 / sizeof(X);              // lanes of a row
            constexpr int RR = L < 32 ? 32 / L : 1;        // rows of an instruction
            const int c = (lane % L) * E;
#pragma unroll 4
            for (int q = L < 32 ? lane / L : 0; q < 32; q += RR)
              if (m0 + q < p.m && n + c < p.n)
                *reinterpret_cast<X*>(static_cast<T*>(p.y) + (m0 + q) * p.n + n + c) = *reinterpret_cast<const X*>(
                    box + q * 64 + (((c / V) ^ ((q >> 1) & 3)) << 4) + (c % V) * sizeof(T));
          };
          const int step = p.n * static_cast<int>(sizeof(T));
          if (step % 8 == 0) by(uint2{});
          else if (sizeof(T) == 4 || step % 4 == 0) by(uint32_t{});
          else if constexpr (sizeof(T) == 2) by(uint16_t{});
          __syncwarp();
        }
      }
    }
    bulk_wait_group0();  // the stores have been performed
  }
  // ---- both CTAs are done (remote arrivals and products too) before the pair frees its TMEM
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

}  // namespace w4a4
