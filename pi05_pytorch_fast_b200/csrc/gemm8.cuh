// Matrix product in 8-bit integers with a scale for each token and each
// output channel:
//   y[m, n] = (sum_k a[m, k] w[n, k]) * sa[m] * sw[n] + bias[n]
// a int8 [m, k] (rows8.cuh), w int8 [n, k].  tcgen05.mma kind::i8 sums exactly
// in int32 (k < 131072), whatever the split; the scaling is fp32, rounded once
// to the output's type.  K is walked in steps of 128 bytes (one 128-byte
// swizzle row); TMA fills what lies past K, M or N with zeros.
//
//  * gemm8_tile_kernel: one tile of 128 channels x T tokens (T <= 256, a
//    multiple of 16) for each cluster of up to 8 CTAs, which split K between
//    them and add their sums through distributed shared memory.  Channels are
//    the MMA's M side, so that few tokens cost few columns.  For one token up
//    to some hundred it is bound by the weights' way from HBM, or by latency.
//  * gemm8_pair_kernel: persistent CTA pairs (cta_group::2), tiles of 256
//    tokens x 256 channels, the accumulators double buffered so that a tile's
//    epilogue runs under the next one's products.  Bound by the tensor pipe.
#pragma once

#include "attention8.cuh"
#include "rows8.cuh"

namespace w4a4 {

struct alignas(64) Gemm8Params {
  CUtensorMap tmap_a;  // tokens: int8 {k, m}, box {128, T or 128}, SW128
  CUtensorMap tmap_w;  // weights: int8 {k, n}, box {128, 128}, SW128
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
  unsigned long long wait_limit_ns;
};

constexpr int kG8StepBytes = 128;             // K bytes of a step
constexpr int kG8ABytes = 128 * kG8StepBytes;  // 16 KB of weights (or tokens) of a step
constexpr int kG8MaxStages = 12;

// (sum of products) -> y: eight consecutive channels of one token.
template <typename T>
__device__ __forceinline__ void g8_store8(const Gemm8Params& p, long long m, int n, const int (&acc)[8], float sa) {
  float v[8];
  T* dst = static_cast<T*>(p.y) + m * p.n + n;
  if (n + 8 <= p.n && p.n % 8 == 0) {
    float w[8];
    load8(p.sw + n, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(acc[i]) * sa * w[i];
    if (p.bias) {
      float b[8];
      load8(static_cast<const T*>(p.bias) + n, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += b[i];
    }
    store8(dst, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < p.n) {
        float x = static_cast<float>(acc[i]) * sa * __ldg(p.sw + n + i);
        if (p.bias) x += to_float(static_cast<const T*>(p.bias)[n + i]);
        dst[i] = from_float<T>(x);
      }
  }
}

__device__ __forceinline__ int4 ld_cluster_i4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// Shared memory: the ring of `stages` (16 KB of weights, T rows of tokens),
// which the sums [T][128] take over once the products are done; barriers.
constexpr int kG8TileThreads = 256;
__host__ __device__ constexpr int gemm8_tile_ring(int tok_tile, int stages) {
  const int ring = stages * (kG8ABytes + tok_tile * kG8StepBytes), sums = tok_tile * 512;
  return ring > sums ? ring : sums;
}
__host__ __device__ constexpr int gemm8_tile_smem(int tok_tile, int stages) {
  const int need = gemm8_tile_ring(tok_tile, stages) + (2 * kG8MaxStages + 1) * 8 + 16 + 1024;
  return need > kOneCtaSmem ? need : kOneCtaSmem;
}

// grid.x = cluster size x token tiles x weight tiles (token tiles fastest, so
// that the CTAs of one weight tile run side by side).
template <typename T>
__global__ void __launch_bounds__(kG8TileThreads) gemm8_tile_kernel(const __grid_constant__ Gemm8Params p) {
  extern __shared__ uint8_t g8_smem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(g8_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  const int S = p.stages, tok_bytes = p.tok_tile * kG8StepBytes;
  uint8_t* w_ring = base;                    // [S][16 KB]
  uint8_t* t_ring = base + S * kG8ABytes;    // [S][T x 128]
  int* sums = reinterpret_cast<int*>(base);  // [T][128], after the products
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + gemm8_tile_ring(p.tok_tile, S));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kG8MaxStages + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const auto bar_full = [&](int s) { return smem_addr(bars + s); };
  const auto bar_empty = [&](int s) { return smem_addr(bars + kG8MaxStages + s); };
  const uint32_t bar_acc = smem_addr(bars + 2 * kG8MaxStages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ranks = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_ctarank());
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
  volatile int no_abort = 0;
  mbar_wait_bounded(bar_acc, 0, &no_abort, err, kErrWaitAccum, limit);
  tc_fence_after();
  __syncthreads();  // the producer has seen its copies land: the ring is free
  // ---- sums to shared memory: lane = channel, so a column's 128 are one line
  const bool aborted = *abort_flag != 0;
  {
    const int quarter = warp & 3;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    for (int c = (warp >> 2) * 16; c < p.tok_tile; c += 32) {
      uint32_t r[16];
      if (steps > 0) {
        tmem_ld_32x32b_x16(tmem_base + lane_addr + c, r);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[(c + j) * 128 + quarter * 32 + lane] = static_cast<int>(r[j]);
    }
  }
  tc_fence_before();
  if (ranks > 1) cluster_sync();
  else __syncthreads();
  // ---- the cluster's CTAs finish a share of the tile each
  const uint32_t sums0 = smem_addr(sums);
  for (int i = rank * kG8TileThreads + threadIdx.x; i < p.tok_tile * 16; i += ranks * kG8TileThreads) {
    const int t = i >> 4, c = (i & 15) * 8;
    const long long m = m0 + t;
    const int n = n0 + c;
    if (m >= p.m || n >= p.n) continue;
    int acc[8] = {};
    for (int r = 0; r < ranks; ++r) {
      const uint32_t at = ranks > 1 ? mapa_shared(sums0 + (t * 128 + c) * 4, r) : sums0 + (t * 128 + c) * 4;
      const int4 x = ld_cluster_i4(at), y = ld_cluster_i4(at + 16);
      acc[0] += x.x, acc[1] += x.y, acc[2] += x.z, acc[3] += x.w;
      acc[4] += y.x, acc[5] += y.y, acc[6] += y.z, acc[7] += y.w;
    }
    if (!aborted) g8_store8<T>(p, m, n, acc, __ldg(p.sa + m));
  }
  if (ranks > 1) cluster_sync();  // no CTA leaves while another may still read its sums
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, cols);
  }
}

// ---------------------------------------------------------------- CTA pairs
// Tiles of 256 tokens (128 in each CTA: the MMA's M side) x 256 channels (128
// weight rows in each CTA's shared memory).  Warp 0 loads, warp 1 of the
// leader issues, warps 2-9 are the epilogue: thread = token row, so a thread
// turns runs of 16 channels into 32-byte stores without shared memory (whose
// bandwidth the products and the copies share).
constexpr int kG8PairStages = 6;
constexpr int kG8PairWarps = 10;
constexpr int kG8PairThreads = 32 * kG8PairWarps;
constexpr int kG8PairSmem = kG8PairStages * 2 * kG8ABytes + 8 * 2 * 128 * 4 + (2 * kG8PairStages + 5) * 8 + 16 + 1024;

// 32 bytes: 16 values of 2 bytes, or 8 of 4.
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void g8_store16(__half* dst, const float (&v)[16]) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = pack_half2_bits(v[2 * i], v[2 * i + 1]);
  st_global_v8(dst, r);
}
__device__ __forceinline__ void g8_store16(__nv_bfloat16* dst, const float (&v)[16]) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    r[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  st_global_v8(dst, r);
}
__device__ __forceinline__ void g8_store16(float* dst, const float (&v)[16]) {
  uint32_t r[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(v[8 * h + i]);
    st_global_v8(dst + 8 * h, r);
  }
}

template <typename T>
__global__ void __launch_bounds__(kG8PairThreads, 1) gemm8_pair_kernel(const __grid_constant__ Gemm8Params p) {
  extern __shared__ uint8_t g8_smem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(g8_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr int S = kG8PairStages;
  uint8_t* t_ring = base;                        // [S][128 tokens x 128]
  uint8_t* w_ring = base + S * kG8ABytes;        // [S][128 weight rows x 128]
  float* chan = reinterpret_cast<float*>(base + 2 * S * kG8ABytes);  // [epilogue warp][scale, bias][128 channels]
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
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    float* sc = chan + (warp - 2) * 256;
    const bool wide = p.n % 16 == 0;
    int count = 0;
    for (int tile = pair; tile < total; tile += n_pairs, ++count) {
      const int buf = count & 1, n0 = tile_n(tile);
      const long long m = tile_m(tile) + row;
      // scales and biases of this warp's four runs of 32 channels, before the sums are ready
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + (2 * j + half) * 32 + lane;
        sc[32 * j + lane] = n < p.n ? __ldg(p.sw + n) : 0.f;
        sc[128 + 32 * j + lane] = p.bias && n < p.n ? to_float(static_cast<const T*>(p.bias)[n]) : 0.f;
      }
      const float sa = m < p.m ? __ldg(p.sa + m) : 0.f;
      __syncwarp();
      if (!warp_all(mbar_wait_bounded_cl(bar_accfull(buf), (count >> 1) & 1, abort_flag, err, kErrWaitAccum, limit))) break;
      tc_fence_after();
      T* dst = static_cast<T*>(p.y) + m * p.n + n0;
      const uint32_t acc = tmem_base + lane_addr + buf * 256;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // 32 columns at a time, alternately by the two warps of a quarter
        const int c = (2 * j + half) * 32;
        uint32_t r[32];
        tmem_ld_32x32b_x16(acc + c, *reinterpret_cast<uint32_t(*)[16]>(&r[0]));
        tmem_ld_32x32b_x16(acc + c + 16, *reinterpret_cast<uint32_t(*)[16]>(&r[16]));
        tmem_ld_wait();
        if (j == 3) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(mapa_shared(bar_accempty(buf), 0));
        }
        if (m >= p.m) continue;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int n = n0 + c + 16 * q;
          if (n >= p.n) continue;
          float v[16];
#pragma unroll
          for (int x = 0; x < 16; x += 4) {
            const float4 w = *reinterpret_cast<const float4*>(sc + 32 * j + 16 * q + x);
            const float4 b = *reinterpret_cast<const float4*>(sc + 128 + 32 * j + 16 * q + x);
            v[x] = fmaf(static_cast<float>(static_cast<int>(r[16 * q + x])) * sa, w.x, b.x);
            v[x + 1] = fmaf(static_cast<float>(static_cast<int>(r[16 * q + x + 1])) * sa, w.y, b.y);
            v[x + 2] = fmaf(static_cast<float>(static_cast<int>(r[16 * q + x + 2])) * sa, w.z, b.z);
            v[x + 3] = fmaf(static_cast<float>(static_cast<int>(r[16 * q + x + 3])) * sa, w.w, b.w);
          }
          if (wide) {
            g8_store16(dst + c + 16 * q, v);
          } else {
#pragma unroll
            for (int x = 0; x < 16; ++x)
              if (n + x < p.n) dst[c + 16 * q + x] = from_float<T>(v[x]);
          }
        }
      }
    }
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
