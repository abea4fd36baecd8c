// Attention of new queries over the 8-bit key/value cache (kv8.cuh).
//
// Query token t of T, head g of the G = H / heads that share key/value head h:
//   S[j] = scale * (q . kc[j]) * ks[j / 16],  P = softmax(S),  O = sum_j P[j] vs[j / 16] vc[j]
// over the keys j < lengths[b] (causal: j < lengths[b] - T + t + 1, the
// queries being the last T tokens of the cache).  A query that sees no key
// gives zeros.
//
// Both kernels work on the rows (t, g) of one key/value head as one matrix:
// the codes go to the tensor cores as fp16 (an int8 is exact in fp16) and the
// block scales are applied outside the products, ks to the scores and vs to
// the probabilities.  Numerics they share:
//  * Q in fp16 times a power of two for each row (bf16 queries keep their 8
//    bits wherever an element is within 2^28 of the row's largest);
//  * scores, row maxima, row sums and O in fp32, softmax in base 2;
//  * a row has two running references.  m is for the sum l of p = 2^(s - m); r
//    is for O, whose weights are w = 2^(s - r) vs, and follows s + e with e the
//    exponent of vs (2^e <= vs < 2^(e+1)), so that it is the row's own largest
//    terms that decide it, whatever the scales of blocks with little weight or
//    of blocks that the row does not see.  Both are set 2^4 above the maximum so
//    far and move only when a block exceeds them by more than 2^11, so that O is
//    rarely rescaled (a rescale of 128 x 256 takes as long as two tiles);
//  * w = p (vs 2^(m - r)) is one exponential a key and one factor a block.  It is
//    rounded to fp16 for the P V product (11 bits, as the scores' own error after
//    exp2 is not much smaller): w < 2^12 fits, the row's largest one is at least
//    2^-4, so what falls below fp16's range is below 2^-20 of it.
// When the keys of a head are split over CTAs, each writes its unnormalised O
// with (m, l) and attn8_join_kernel adds them up.
#pragma once

#include "attention.cuh"
#include "kv8.cuh"

namespace w4a4 {

// At least 160 KB of shared memory for a CTA with TMEM, so that no other one of
// this library shares its SM, the 4-bit products with their narrowest tiles (71 KB)
// among them.  A CTA that waits for columns waits without a limit, and could for
// good: two clusters (of two streams), each with one half's columns taken by the
// other; or a kernel that has let its dependents start and asks for its columns
// only then, which a dependent holds until that kernel is over.
constexpr int kOneCtaSmem = 160 * 1024;
constexpr float kAttn8Margin = 4.f;    // log2 by which m and r are set above a row's maxima
constexpr float kAttn8Grow = 11.f;     // log2 by which a block may exceed them

struct Attn8Params {
  const void* q;  // [batch, tokens, q_heads, width]
  void* out;      // contiguous
  const int8_t* k;
  const int8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* lengths;
  float* part_o;           // [batch * heads][splits][rows][width], 16-byte chunk c of row r at c ^ (r & 7)
  float2* part_ml;         // [batch * heads][splits][rows]
  long long qb, qt, qh;    // query strides (elements)
  long long cb, ct, ch;    // cache strides
  int tokens, heads, group, capacity;  // group: query heads of a key/value head
  int rows;                // tokens * group
  int splits;
  int causal;
  float scale;             // softmax scale * log2(e)
  unsigned long long wait_limit_ns;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two of four codes, given as code + 128 in the bytes of w, as fp16: 0x6400 |
// u is 1024 + u, so subtracting 1152 leaves the code, exactly.
template <int HI>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t w) {
  const uint32_t u = __byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// D (16 x 8, fp32) += A (16 x 16, fp16) B (16 x 8, fp16).
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr float kMaxFloat = 3.4028234e38f;

// The exponent of a value scale; none (-infinity) for zero, and for one that is
// not finite, whose rows are not finite whatever the reference.
__device__ __forceinline__ float value_exponent(float vs) {
  const float e = __uint_as_float(0x4b000000u | (__float_as_uint(vs) >> 23)) - (8388608.f + 127.f);
  return vs > 0.f && vs <= kMaxFloat ? e : -INFINITY;
}
// 2^(d / 2): half of the way from one reference to another, as the whole of it
// may leave fp32's range where its product with a scale does not.
__device__ __forceinline__ float half_way(float d) { return fminf(ex2_approx(0.5f * d), 8.507059e37f); }  // 2^126
// What turns p into w: vs 2^(m - r), `half` being half_way(m - r).  Past fp32's range
// p is zero.
__device__ __forceinline__ float value_factor(float vs, float half) { return fminf(vs * half * half, kMaxFloat); }
__device__ __forceinline__ float any_value_factor(float vs, float half) {
  return vs <= kMaxFloat ? value_factor(vs, half) : __uint_as_float(0x7fc00000u);
}
// p times that; keys that are not seen (p = 0) add nothing whatever it is.
__device__ __forceinline__ float weigh(float p, float factor) { return p == 0.f ? 0.f : p * factor; }

// The power of two by which a row of queries is multiplied so that its largest
// element lies in [2^14, 2^15) of fp16 (1 for a zero row).
__device__ __forceinline__ float query_shift(float amax) {
  const int e = static_cast<int>(__float_as_uint(amax) >> 23);  // biased exponent
  if (e == 0) return amax == 0.f ? 1.f : 1.7014118e38f;         // subnormal: 2^127
  return __uint_as_float(static_cast<uint32_t>(max(1, min(254, 254 - e + 14))) << 23);  // 2^(127 - e + 14)
}

// Keys seen by query token t of an observation with n tokens in its cache.
__device__ __forceinline__ int keys_seen(const Attn8Params& p, int n, int t) {
  return p.causal ? max(0, n - p.tokens + t + 1) : n;
}

// ------------------------------------------------------- few rows (<= 16)
// The form for single tokens.  The warps of all CTAs of one key/value head
// (splits x kWarps) take its steps of 256 / D blocks of 16 keys in turn, each
// on its own, through its own ring of cp.async stages of 8 KB, with mma.sync
// m16n8k16: the 16 rows are the heads of the group, so a block's K and V are
// read once for all of them.  The K index of an MMA may be permuted freely
// when both operands agree, and so may the columns of V; so every lane reads
// 16 consecutive bytes:
//  * K: lane (g, t) of a key row g holds dims 64 c + 16 t ... + 15 = four steps
//    of four dims, and Q's fragments are kept in the same order;
//  * V: lane (g, t) holds dims 16 g ... + 15 of the keys 2t, 2t+1, 2t+8, 2t+9;
//    pairs of keys are zipped with byte permutes; column n of tile e is dim
//    16 n + e, so a lane ends with runs of 16 consecutive dims of O.
// w goes in as the sum of two fp16, its rounding and the rest: with at most 8
// rows (HALF) the rest takes the idle rows 8-15 of the same MMA, with more it
// is a second one.  The four lanes of a row agree on r (O's columns are theirs
// in turns); m and l are each lane's own until the end.  Bound: HBM (2 width bytes per key); legacy MMA is enough
// for it.  Which warp takes which keys does not depend on the lengths, so the
// first loads are under way before the length has arrived.  Measured: 8 heads of
// 256 over 776 tokens 7.4 us, over 131,072 (67 MB) 26.3 us; 4 x 16 heads on 2 of 128
// over 65,536 (134 MB) 33 to 34 us: 5.4 to 6 TB/s once it streams.
template <int D, bool HALF>
struct Attn8Few {
  static constexpr int kWarps = 8, kStages = 3;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kRowsMax = HALF ? 8 : 16;
  static constexpr int kBlocks = 256 / D;           // token blocks of a step
  static constexpr int kChunks = D / 16;            // 16-byte chunks of a key
  static constexpr int kHalfStage = kKvBlock * 256; // K or V of a step
  static constexpr int kStage = 2 * kHalfStage + 64;  // K, V, scales
  static constexpr int kRing = kStages * kStage;    // of a warp
  static constexpr int kPad = D + 4;                // row of the O exchange (floats)
  static constexpr int kQBytes = 16 * D * 2;
  static constexpr int kExchange = (kWarps + 1) * kRowsMax * kPad * 4;  // in the rings, when they are idle
  static constexpr int kSmem = kQBytes + 16 * 8 + (kWarps + 1) * kRowsMax * 8 + kWarps * kRing;
  static_assert(kExchange <= kWarps * kRing, "the exchange must fit the rings");
  // byte offset of 16-byte chunk c of key row r: swizzled so that the reads below hit every bank once
  __device__ static __forceinline__ int k_at(int r, int c) {
    const int l = r * kChunks + c;
    return 16 * (D >= 128 ? l ^ ((r & 1) << 2) : l);
  }
  __device__ static __forceinline__ int v_at(int r, int c) { return 16 * ((r * kChunks + c) ^ (((r >> 1) & 3) << 1)); }
};

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// 4 consecutive results, rounded once.
template <typename T>
__device__ __forceinline__ void store4(T* dst, const float4& v) {
  if constexpr (std::is_same_v<T, float>) {
    *reinterpret_cast<float4*>(dst) = v;
  } else if constexpr (std::is_same_v<T, __half>) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_half2_bits(v.x, v.y), pack_half2_bits(v.z, v.w));
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
}
// Row r of a key/value head's rows (unit = batch x heads) in the output.
__device__ __forceinline__ long long out_row(const Attn8Params& p, int b, int h, int r) {
  return (static_cast<long long>(b) * p.tokens + r / p.group) * (p.heads * p.group) + h * p.group + r % p.group;
}

template <typename T, int D, bool HALF>
__global__ void __launch_bounds__(Attn8Few<D, HALF>::kThreads, 1)
    attn8_few_kernel(const __grid_constant__ Attn8Params p) {
  using C = Attn8Few<D, HALF>;
  extern __shared__ __align__(128) uint8_t few_smem[];
  uint8_t* q_smem = few_smem;                                        // fp16 [16][D], chunk c of row r at c ^ (r & 1)
  float2* row_info = reinterpret_cast<float2*>(q_smem + C::kQBytes); // score factor, keys seen
  float2* warp_ml = row_info + 16;                                   // [warps + 1][rows]; the last is the CTA's
  uint8_t* rings = reinterpret_cast<uint8_t*>(warp_ml + (C::kWarps + 1) * C::kRowsMax);
  float* xo = reinterpret_cast<float*>(rings);                       // [warps + 1][rows][kPad], after the last step
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, unit = blockIdx.y;
  const int b = unit / p.heads, h = unit - b * p.heads;
  pdl_launch_dependents();
  pdl_wait();
  const int8_t* kc = p.k + b * p.cb + h * p.ch;
  const int8_t* vc = p.v + b * p.cb + h * p.ch;
  const int blocks = p.capacity / kKvBlock;
  const float* ks = p.ks + static_cast<long long>(unit) * blocks;
  const float* vs = p.vs + static_cast<long long>(unit) * blocks;
  constexpr int KC = D / 64;                   // 64-dim chunks of a key
  constexpr int VU = D >= 128 ? D / 128 : 1;   // runs of dims of a lane
  constexpr int VW = D >= 128 ? 4 : 2;         // words of a run
  constexpr int NB = C::kBlocks;
  uint8_t* ring = rings + warp * C::kRing;
  // a step's keys, values and scales into a stage (every slot of a block exists, the capacity being a multiple of 16)
  const auto fetch = [&](int step, int stage) {
    const uint32_t dst = smem_addr(ring) + stage * C::kStage;
    const int blk = step * NB;
    const int rows = min(blocks - blk, NB) * kKvBlock;
    const int r0 = lane / C::kChunks, c = lane % C::kChunks;
    const long long at = (static_cast<long long>(blk) * kKvBlock + r0) * p.ct + 16 * c;
    const int8_t* kb = kc + at;
    const int8_t* vb = vc + at;
    constexpr int kStep = 32 / C::kChunks;  // rows of a warp's instruction
#pragma unroll
    for (int i = 0; i < kKvBlock * NB / kStep; ++i) {
      const int r = r0 + kStep * i;
      if (NB == 1 || r < rows) {
        cp_async16(dst + C::k_at(r, c), kb + i * kStep * p.ct);
        cp_async16(dst + C::kHalfStage + C::v_at(r, c), vb + i * kStep * p.ct);
      }
    }
    if (lane < 2 * NB && blk + (lane >> 1) < blocks)
      cp_async4(dst + 2 * C::kHalfStage + 4 * lane, (lane & 1 ? vs : ks) + blk + (lane >> 1));
  };
  const int stride = p.splits * C::kWarps;
  int step = split * C::kWarps + warp;
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) {
    if ((step + i * stride) * NB < blocks) fetch(step + i * stride, i);
    cp_async_commit();
  }
  const int n = min(max(p.lengths[b], 0), p.capacity);
  const int nblk = (n + kKvBlock - 1) / kKvBlock;
  const int nsteps = (nblk + NB - 1) / NB;
  {
    // Q: 16 threads per row, D / 16 consecutive elements each
    constexpr int E = D / 16;
    const int r = threadIdx.x >> 4, e0 = (threadIdx.x & 15) * E;
    float v[E];
    uint32_t key = 0;
    const int tok = r / p.group, head = h * p.group + r % p.group;
    const T* src = static_cast<const T*>(p.q) + b * p.qb + tok * p.qt + head * p.qh + e0;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = 0.f;
    if (r < p.rows) {
      if constexpr (E >= 8) {
#pragma unroll
        for (int i = 0; i < E; i += 8) load8(src + i, *reinterpret_cast<float(*)[8]>(&v[i]));
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = to_float(src[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) key = max(key, abs_key(v[i]));
#pragma unroll
    for (int o = 8; o; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    const float shift = query_shift(__uint_as_float(key));
    const float up = p.scale < 0.f ? -shift : shift;  // the factor below is not negative
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const int e = e0 + i;
      *reinterpret_cast<uint32_t*>(q_smem + r * 2 * D + ((((e >> 3) ^ (r & 1)) << 4) | ((e & 7) * 2))) =
          pack_half2_bits(v[i] * up, v[i + 1] * up);
    }
    if ((threadIdx.x & 15) == 0)
      row_info[r] = make_float2(fabsf(p.scale) / shift, __int_as_float(r < p.rows ? keys_seen(p, n, tok) : 0));
  }
  __syncthreads();
  constexpr int R = HALF ? 1 : 2;  // rows g, g + 8 of a lane
  float factor[R], m[R], l[R], ref[R];
  int seen[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float2 info = row_info[g + 8 * i];
    factor[i] = info.x;
    seen[i] = __float_as_int(info.y);
    m[i] = ref[i] = -INFINITY;
    l[i] = 0.f;
  }
  float o[D / 8][4];
#pragma unroll
  for (int e = 0; e < D / 8; ++e) o[e][0] = o[e][1] = o[e][2] = o[e][3] = 0.f;

  int stage = 0;
  for (; step < nsteps; step += stride) {
    cp_async_wait<C::kStages - 2>();
    __syncwarp();
    {
      const int next = step + stride * (C::kStages - 1);
      if (next < nsteps) fetch(next, stage == 0 ? C::kStages - 1 : stage - 1);
      cp_async_commit();
    }
    const uint8_t* kt = ring + stage * C::kStage;
    const uint8_t* vt = kt + C::kHalfStage;
    const float2* sc = reinterpret_cast<const float2*>(vt + C::kHalfStage);
    stage = stage + 1 == C::kStages ? 0 : stage + 1;
    // ---- S (rows x 16 NB keys): tile 2q + i has keys 16q + 8i + 2t, + 1
    float s[2 * NB][4] = {};
    float s2[NB == 1 ? 2 : 1][4] = {};  // D = 256: a second accumulator halves the chain of dependent products
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      uint32_t qa[8], qb[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = ((8 * c + 2 * t + u) ^ (g & 1)) << 4;
        *reinterpret_cast<uint4*>(&qa[4 * u]) = *reinterpret_cast<const uint4*>(q_smem + g * 2 * D + at);
        if constexpr (!HALF)
          *reinterpret_cast<uint4*>(&qb[4 * u]) = *reinterpret_cast<const uint4*>(q_smem + (g + 8) * 2 * D + at);
        else
          qb[4 * u] = qb[4 * u + 1] = qb[4 * u + 2] = qb[4 * u + 3] = 0u;
      }
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        const uint4 k = *reinterpret_cast<const uint4*>(kt + C::k_at(8 * i + g, 4 * c + t));
        const uint32_t w[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t u = w[x] ^ 0x80808080u;
          mma_16816(NB == 1 && (x & 1) ? s2[i & 1] : s[i], qa[2 * x], qb[2 * x], qa[2 * x + 1], qb[2 * x + 1],
                    codes_to_half2<0>(u), codes_to_half2<1>(u));
        }
      }
    }
    if constexpr (NB == 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] += s2[i][j];
    }
    // ---- softmax of the step
    const int j0 = step * NB * kKvBlock + 2 * t;
    float vsc[NB];
    float bm[R], br[R];  // maxima of s, and of s + e
#pragma unroll
    for (int i = 0; i < R; ++i) bm[i] = br[i] = -INFINITY;
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      const bool has = step * NB + q < nblk;  // past the length: what the stage holds is not a scale
      const float2 x = sc[q];
      vsc[q] = has ? x.y : 0.f;
      const float e = value_exponent(vsc[q]);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float fk = has ? factor[i] * x.x : 0.f;
        const int left = seen[i] - j0 - 16 * q;
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float& v = s[2 * q + (j >> 1)][2 * i + (j & 1)];
          v = (j & 1) + 8 * (j >> 1) < left ? v * fk : -INFINITY;
          top = fmaxf(top, v);
        }
        bm[i] = fmaxf(bm[i], top);
        br[i] = fmaxf(br[i], top + e);
      }
    }
    float f[R], half[R];
    bool grow = false;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (bm[i] > m[i] + kAttn8Grow) {
        bm[i] += kAttn8Margin;
        l[i] *= m[i] == -INFINITY ? 0.f : ex2_approx(m[i] - bm[i]);
        m[i] = bm[i];
      }
      br[i] = fmaxf(br[i], __shfl_xor_sync(0xffffffffu, br[i], 1));
      br[i] = fmaxf(br[i], __shfl_xor_sync(0xffffffffu, br[i], 2));
      f[i] = 1.f;
      if (br[i] > ref[i] + kAttn8Grow) {
        br[i] += kAttn8Margin;
        f[i] = ref[i] == -INFINITY ? 0.f : ex2_approx(ref[i] - br[i]);
        ref[i] = br[i];
        grow = true;
      }
      half[i] = half_way(m[i] - ref[i]);
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int e = 0; e < D / 8; ++e)
#pragma unroll
        for (int i = 0; i < R; ++i) {
          o[e][2 * i] *= f[i];
          o[e][2 * i + 1] *= f[i];
          if constexpr (HALF) {  // rows 8-15 hold what the rest of w adds to rows 0-7
            o[e][2] *= f[0];
            o[e][3] *= f[0];
          }
        }
    }
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      uint32_t ph[R][2], pl[R][2];  // w and the rest of its rounding: [rows][keys]
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float nm = m[i] == -INFINITY ? 0.f : -m[i];
        const float rv = any_value_factor(vsc[q], half[i]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float p0 = ex2_approx(s[2 * q + j][2 * i] + nm), p1 = ex2_approx(s[2 * q + j][2 * i + 1] + nm);
          l[i] += p0 + p1;
          const float w0 = weigh(p0, rv), w1 = weigh(p1, rv);
          const __half2 hi = __floats2half2_rn(w0, w1);
          const float2 back = __half22float2(hi);
          ph[i][j] = *reinterpret_cast<const uint32_t*>(&hi);
          pl[i][j] = pack_half2_bits(w0 - back.x, w1 - back.y);
        }
      }
      // ---- O += P V
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        uint32_t vr[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * q + 2 * t + (i & 1) + 8 * (i >> 1);
          if constexpr (VW == 4)
            *reinterpret_cast<uint4*>(vr[i]) = *reinterpret_cast<const uint4*>(vt + C::v_at(r, g + 8 * u));
          else
            *reinterpret_cast<uint2*>(vr[i]) = *reinterpret_cast<const uint2*>(vt + C::v_at(r, g >> 1) + 8 * (g & 1));
        }
#pragma unroll
        for (int x = 0; x < VW; ++x) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = vr[i][x] ^ 0x80808080u;
          // keys (2t, 2t + 1) and (2t + 8, 2t + 9) of dims 4x .. 4x + 3, two dims a word
          const uint32_t z[4] = {__byte_perm(w[0], w[1], 0x5140), __byte_perm(w[2], w[3], 0x5140),
                                 __byte_perm(w[0], w[1], 0x7362), __byte_perm(w[2], w[3], 0x7362)};
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float(&d0)[4] = o[u * 16 + 4 * x + 2 * y];
            float(&d1)[4] = o[u * 16 + 4 * x + 2 * y + 1];
            const uint32_t b0 = codes_to_half2<0>(z[2 * y]), b1 = codes_to_half2<0>(z[2 * y + 1]);
            const uint32_t c0 = codes_to_half2<1>(z[2 * y]), c1 = codes_to_half2<1>(z[2 * y + 1]);
            if constexpr (HALF) {
              mma_16816(d0, ph[0][0], pl[0][0], ph[0][1], pl[0][1], b0, b1);
              mma_16816(d1, ph[0][0], pl[0][0], ph[0][1], pl[0][1], c0, c1);
            } else {
              mma_16816(d0, ph[0][0], ph[R - 1][0], ph[0][1], ph[R - 1][1], b0, b1);
              mma_16816(d1, ph[0][0], ph[R - 1][0], ph[0][1], ph[R - 1][1], c0, c1);
              mma_16816(d0, pl[0][0], pl[R - 1][0], pl[0][1], pl[R - 1][1], b0, b1);
              mma_16816(d1, pl[0][0], pl[R - 1][0], pl[0][1], pl[R - 1][1], c0, c1);
            }
          }
        }
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // every warp has left its ring
  // ---- the CTA's warps: O, m and l of each through shared memory
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float top = fmaxf(m[i], __shfl_xor_sync(0xffffffffu, m[i], 1));  // the row's m, from its lanes'
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    l[i] *= m[i] == -INFINITY ? 1.f : ex2_approx(m[i] - top);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (t == 0) warp_ml[warp * C::kRowsMax + g + 8 * i] = make_float2(top, l[i]);
    const float back = top == -INFINITY ? 0.f : half_way(ref[i] - top);  // O as the others' will be: with 2^-m
    float* row = xo + (warp * C::kRowsMax + g + 8 * i) * C::kPad;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int e = 0; e < D / 8; e += 4) {
        constexpr int run = D >= 128 ? 16 : 8;
        const int dim = (e / 16) * 128 + (2 * t + half) * run + e % 16;
        float4 x;
        float* xs = &x.x;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          xs[j] = (HALF ? o[e + j][half] + o[e + j][2 + half] : o[e + j][2 * i + half]) * back * back;
        *reinterpret_cast<float4*>(row + dim) = x;
      }
  }
  __syncthreads();
  const int ranks = static_cast<int>(cluster_nctarank());
  const bool direct = p.splits == 1;          // this CTA has all the keys
  const bool clustered = !direct && ranks == p.splits;
  const int items = p.rows * (D / 4);
  for (int i = threadIdx.x; i < items; i += C::kThreads) {
    const int r = i / (D / 4), e = (i - r * (D / 4)) * 4;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) mm = fmaxf(mm, warp_ml[w * C::kRowsMax + r].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) {
      const float2 ml = warp_ml[w * C::kRowsMax + r];
      if (ml.y == 0.f) continue;  // saw nothing (a NaN stays)
      const float f = ex2_approx(ml.x - mm);
      const float4 x = *reinterpret_cast<const float4*>(xo + (w * C::kRowsMax + r) * C::kPad + e);
      acc.x = fmaf(x.x, f, acc.x), acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z), acc.w = fmaf(x.w, f, acc.w);
      sum = fmaf(ml.y, f, sum);
    }
    if (direct) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      store4(static_cast<T*>(p.out) + out_row(p, b, h, r) * D + e,
             make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    } else if (clustered) {
      *reinterpret_cast<float4*>(xo + (C::kWarps * C::kRowsMax + r) * C::kPad + e) = acc;
      if (e == 0) warp_ml[C::kWarps * C::kRowsMax + r] = make_float2(mm, sum);
    } else {
      const long long at = (static_cast<long long>(unit) * p.splits + split) * p.rows + r;
      *reinterpret_cast<float4*>(p.part_o + at * D + ((e / 4) ^ (r & 7)) * 4) = acc;
      if (e == 0) p.part_ml[at] = make_float2(mm, sum);
    }
  }
  if (clustered) {
    // ---- the cluster's CTAs: each finishes its share of the results, reading the others' shared memory
    cluster_sync();
    const uint32_t ml0 = smem_addr(warp_ml + C::kWarps * C::kRowsMax), xo0 = smem_addr(xo + C::kWarps * C::kRowsMax * C::kPad);
    for (int i = split * C::kThreads + threadIdx.x; i < items; i += ranks * C::kThreads) {
      const int r = i / (D / 4), e = (i - r * (D / 4)) * 4;
      float2 ml[8];
      float4 x[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if (c >= ranks) break;
        ml[c] = ld_cluster_v2(mapa_shared(ml0 + r * 8, c));
        x[c] = ld_cluster_v4(mapa_shared(xo0 + (r * C::kPad + e) * 4, c));
      }
      float mm = -INFINITY;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < ranks) mm = fmaxf(mm, ml[c].x);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if (c >= ranks || ml[c].y == 0.f) continue;
        const float f = ex2_approx(ml[c].x - mm);
        acc.x = fmaf(x[c].x, f, acc.x), acc.y = fmaf(x[c].y, f, acc.y);
        acc.z = fmaf(x[c].z, f, acc.z), acc.w = fmaf(x[c].w, f, acc.w);
        sum = fmaf(ml[c].y, f, sum);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      store4(static_cast<T*>(p.out) + out_row(p, b, h, r) * D + e,
             make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
    cluster_sync();  // no CTA leaves while another may still read its shared memory
  }
}

// ------------------------------------------------------ many rows (> 16)
// tcgen05: a CTA takes 128 rows (t, g) of one key/value head and a range of
// its keys, in tiles of 64.  Q lies in TMEM, as the A operand of S = Q K^T (from
// shared memory its reads alone would take the products' time again).  The
// codes come by TMA and become fp16 in shared memory once per tile and CTA, by
// eight warps of their own:
//   warps 0-7    softmax and epilogue (thread = row = TMEM lane): warps 0-3 take
//                the even tiles, 4-7 the odd ones, so that one group's
//                exponentials run beside the other's maxima; each has its own m
//                and l, and r passes from tile to tile through shared memory
//   warps 8-11   keys: 16 codes a load -> K-major rows, 128-byte swizzle
//   warps 12-15  values: 8 keys of up to 16 dims -> V^T rows of 64 keys (byte
//                permutes), as the second product wants its B operand K-major
//   warp 16      issues S = Q K^T (M 128, N 64) and O += P V (M 128, N D)
//   warp 17      asks for the codes (TMA, two tiles ahead)
// Codes, K and V^T tiles and P are double buffered; the one score buffer is
// free again as soon as its readers have it in registers, so S(i + 2) is under
// way before P(i) V; O stays in TMEM.  Keys sit in a tile in the order rho =
// 8 (j % 8) + j / 8: an eighth of the tile's keys lies 8 rows apart in the codes,
// where the swizzle spreads them over all banks.
// setmaxnreg moves registers to the softmax warps (of 640 x 96: 256 x 128 for
// them, 256 x 80 for the converters, 128 x 56 for the rest).
// At D = 256 a tile costs the tensor pipe 1024 cycles, shared memory 1280 (codes
// read, fp16 written, operands read) and the exponentials (16 a cycle) 512;
// measured are 3080 (512 tokens x 8 heads over 16,384: 114 to 118 us, tensor pipe
// 38 %), 2120 at D = 128 and 1930 at D = 64: the chain of a tile is what bounds it.
template <int D>
struct Attn8Many {
  static constexpr int kRows = 128, kKeys = 64;
  static constexpr int kSlices = D / 64;
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kKBytes = kKeys * D * 2, kVBytes = D * kKeys * 2, kRaw = kKeys * D;
  static constexpr int kSoftWarps = 8, kThreads = 20 * 32;
  static constexpr int kSoftRegs = 128, kConvRegs = 80, kRestRegs = 56;
  static constexpr int kPoolRegs = 256 * kSoftRegs + 256 * kConvRegs + 128 * kRestRegs;
  static constexpr int kNumBars = 33;
  // K and V^T rings (the raw Q before, and O after the tiles, use them), rings of codes, row data: score factor, keys
  // seen; l of both groups; r; m of both groups
  static constexpr int kRing = 2 * (kKBytes + kVBytes);
  static constexpr int kNeed = kRing + 4 * kRaw + kRows * 8 + 5 * kRows * 4 + kNumBars * 8 + 32 + 1024;
  static constexpr uint32_t kTmemCols = D == 64 ? 256 : 512;
  static constexpr int kSmem = kNeed > kOneCtaSmem ? kNeed : kOneCtaSmem;
  static constexpr uint32_t kOCol = 0, kQCol = D, kSCol = D == 64 ? 128 : D + D / 2, kPCol = kSCol + kKeys;
  static_assert(2 * kKBytes >= kQBytes && kRing >= kRows * D * 4, "Q and O must fit the rings");
};

struct alignas(64) Attn8ManyParams {
  CUtensorMap tmap_k, tmap_v;  // int8 {width, heads, capacity, batch}, box {min(width, 128), 1, 64, 1}, swizzle = its width
  Attn8Params p;
};

__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(Attn8Many<D>::kThreads, 1)
    attn8_many_kernel(const __grid_constant__ Attn8ManyParams params) {
  using C = Attn8Many<D>;
  const Attn8Params& p = params.p;
  extern __shared__ uint8_t many_smem[];
  uint8_t* base =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(many_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* k_ring = base;                       // [2][slices][64 rows][128 B]
  uint8_t* q_smem = base;                       // (before) [128 rows][2 D B], 16-byte chunk c of row r at c ^ (r & 7)
  uint8_t* v_ring = k_ring + 2 * C::kKBytes;    // [2][D rows][128 B]
  uint8_t* k_raw = v_ring + 2 * C::kVBytes;     // [2][D / 128 (at least 1) boxes][64 keys][128 or 64 B]
  uint8_t* v_raw = k_raw + 2 * C::kRaw;
  float2* row_info = reinterpret_cast<float2*>(v_raw + 2 * C::kRaw);      // score factor, keys seen
  float* row_x = reinterpret_cast<float*>(row_info + C::kRows);           // [2 groups][128 rows]: amax of half of Q, later l
  float* row_r = row_x + 2 * C::kRows;                                    // running references of O
  float* row_m = row_r + C::kRows;                                        // [2 groups][128 rows]: m, after the tiles
  uint64_t* bars = reinterpret_cast<uint64_t*>(row_m + 2 * C::kRows);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* plan = reinterpret_cast<int*>(tmem_slot + 2);  // length, first tile, tiles
  const auto bar_kraw = [&](int s) { return smem_addr(bars + s); };        // codes landed
  const auto bar_vraw = [&](int s) { return smem_addr(bars + 2 + s); };
  const auto bar_kread = [&](int s) { return smem_addr(bars + 4 + s); };   // codes read
  const auto bar_vread = [&](int s) { return smem_addr(bars + 6 + s); };
  const auto bar_kfull = [&](int s) { return smem_addr(bars + 8 + s); };
  const auto bar_kempty = [&](int s) { return smem_addr(bars + 10 + s); };
  const auto bar_vfull = [&](int s) { return smem_addr(bars + 12 + s); };
  const auto bar_vempty = [&](int s) { return smem_addr(bars + 14 + s); };
  const auto bar_pfull = [&](int s) { return smem_addr(bars + 16 + s); };
  const auto bar_pfree = [&](int s) { return smem_addr(bars + 18 + s); };  // P V of that parity's last tile is done
  const auto bar_r = [&](int q) { return smem_addr(bars + 20 + q); };      // a quarter's references of a tile are decided
  const auto bar_l = [&](int q) { return smem_addr(bars + 24 + q); };      // both groups' sums of a quarter are there
  // one for each group, as a wait for a phase must not begin before the phase before it has passed
  const auto bar_sfull = [&](int s) { return smem_addr(bars + 28 + s); };
  const uint32_t bar_sread = smem_addr(bars + 30), bar_o = smem_addr(bars + 31), bar_q = smem_addr(bars + 32);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.y, unit = blockIdx.z;
  const int b = unit / p.heads, h = unit - b * p.heads;
  const int r0 = blockIdx.x * C::kRows;
  unsigned* err = &g_w4a4_device_error;
  const uint64_t limit = p.wait_limit_ns;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_kraw(s), 1);
      mbar_init(bar_vraw(s), 1);
      mbar_init(bar_kread(s), 4);
      mbar_init(bar_vread(s), 4);
      mbar_init(bar_kfull(s), 4);
      mbar_init(bar_kempty(s), 1);
      mbar_init(bar_vfull(s), 4);
      mbar_init(bar_vempty(s), 1);
      mbar_init(bar_pfull(s), 4);
      mbar_init(bar_pfree(s), 1);
      mbar_init(bar_sfull(s), 1);
    }
    for (int q = 0; q < 4; ++q) {
      mbar_init(bar_r(q), 1);
      mbar_init(bar_l(q), 2);
    }
    mbar_init(bar_sread, 4);
    mbar_init(bar_o, 1);
    mbar_init(bar_q, C::kSoftWarps);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 16) {
    tmem_alloc(smem_addr(tmem_slot), C::kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  constexpr int QC = D * 2 / 16;  // 16-byte chunks of a row of Q
  if (warp < C::kSoftWarps) {
    // Q as it comes to shared memory; a lane works out where one of the warp's 16 rows is
    const int ri = r0 + warp + C::kSoftWarps * (lane & 15);
    const int tok = ri / p.group, g = ri - tok * p.group;
    const long long off = b * p.qb + tok * p.qt + (h * p.group + g) * p.qh;
#pragma unroll 2
    for (int i = 0; i < 16; ++i) {
      const int x = warp + C::kSoftWarps * i;
      const long long o = __shfl_sync(0xffffffffu, off, i);
      const uint32_t dst = smem_addr(q_smem) + x * 2 * D + ((lane ^ (x & 7)) << 4);
      if (lane < QC) {
        if (r0 + x < p.rows) cp_async16(dst, static_cast<const T*>(p.q) + o + lane * 8);
        else asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0u) : "memory");
      }
    }
    cp_async_commit();
  } else if (threadIdx.x == 17 * 32) {
    // which tiles: the keys that the last row sees (an earlier row never sees more), this split's share
    const int len = min(max(p.lengths[b], 0), p.capacity);
    const int last = min(p.rows, r0 + C::kRows) - 1;
    const int tiles = (keys_seen(p, len, p.causal ? last / p.group : 0) + C::kKeys - 1) / C::kKeys;
    const int per = (tiles + p.splits - 1) / p.splits;
    const int first = min(tiles, split * per);
    plan[0] = len;
    plan[1] = first;
    plan[2] = min(tiles, first + per) - first;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int n = plan[0], tile0 = plan[1], nt = plan[2];
  const int nblocks = (n + kKvBlock - 1) / kKvBlock;  // blocks with a scale

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRestRegs));
    if (warp == 17) {
      // ---------------------------------------------- codes (lane 0)
      if (lane == 0) {
        constexpr int kBoxes = D > 128 ? D / 128 : 1, kBox = C::kRaw / kBoxes;
        int issued = 0;
        for (int i = 0; i < nt; ++i, ++issued) {
          const int slot = i & 1, j0 = (tile0 + i) * C::kKeys;
          if (i >= 2 && !mbar_wait_spin(bar_kread(slot), ((i >> 1) - 1) & 1, abort_flag, err, kErrWaitEmpty, limit)) break;
          mbar_arrive_expect_tx(bar_kraw(slot), C::kRaw);
          for (int x = 0; x < kBoxes; ++x)
            tma_load_4d(smem_addr(k_raw + slot * C::kRaw + x * kBox), &params.tmap_k, 128 * x, h, j0, b, bar_kraw(slot));
          if (i >= 2 && !mbar_wait_spin(bar_vread(slot), ((i >> 1) - 1) & 1, abort_flag, err, kErrWaitEmpty, limit)) {
            volatile int no_abort = 0;
            mbar_wait_bounded(bar_kraw(slot), (i >> 1) & 1, &no_abort, err, kErrWaitDrain, limit);
            break;
          }
          mbar_arrive_expect_tx(bar_vraw(slot), C::kRaw);
          for (int x = 0; x < kBoxes; ++x)
            tma_load_4d(smem_addr(v_raw + slot * C::kRaw + x * kBox), &params.tmap_v, 128 * x, h, j0, b, bar_vraw(slot));
        }
        // no copy may still be in flight at exit
        volatile int no_abort = 0;
        for (int i = max(0, issued - 2); i < issued; ++i) {
          mbar_wait_bounded(bar_kraw(i & 1), (i >> 1) & 1, &no_abort, err, kErrWaitDrain, limit);
          mbar_wait_bounded(bar_vraw(i & 1), (i >> 1) & 1, &no_abort, err, kErrWaitDrain, limit);
        }
      }
      __syncwarp();
    } else if (warp == 16) {
      // ---------------------------------------------- MMA issuer (one elected lane)
      const bool issuer = elect_one();
      const uint32_t idesc_s = idesc_f16(C::kRows, C::kKeys);
      const uint32_t idesc_o = idesc_f16(C::kRows, D);
      bool alive = nt == 0 || warp_all(mbar_wait_spin(bar_q, 0, abort_flag, err, kErrWaitUnpack, limit));
      // whichever product is ready next: S(si) (its keys are there and S(si - 1) has been read) or P(pi) V.  S(si) comes
      // after P(si - 3) V, so that bar_sfull(si) covers it too: the group of tile si may wait for P(si - 1) V, by parity
      // on the other group's barrier, and must know the phase before that one to be over
      int si = 0, pi = 0, idle = 0;
      uint64_t since = 0;
      while (alive && pi < nt) {
        const int ss = si & 1, ps = pi & 1;
        const bool s_ready = si < nt && si <= pi + 2 && mbar_test_wait(bar_kfull(ss), (si >> 1) & 1) &&
                             (si == 0 || mbar_test_wait(bar_sread, (si - 1) & 1));
        if (__any_sync(0xffffffffu, s_ready)) {
          tc_fence_after();
          const uint64_t kdesc = smem_desc_sw128(smem_addr(k_ring + ss * C::kKBytes));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            if (issuer)
              umma_f16_ts(tmem_base + C::kSCol, tmem_base + C::kQCol + 8 * kk,
                          kdesc + static_cast<uint64_t>((kk >> 2) * (C::kKeys * 128) >> 4) + static_cast<uint64_t>((kk & 3) * 2),
                          idesc_s, kk > 0);
          if (issuer) {
            umma_commit(bar_sfull(ss));
            umma_commit(bar_kempty(ss));
          }
          __syncwarp();
          ++si;
          idle = 0;
          continue;
        }
        const bool p_ready = mbar_test_wait(bar_vfull(ps), (pi >> 1) & 1) && mbar_test_wait(bar_pfull(ps), (pi >> 1) & 1);
        if (__any_sync(0xffffffffu, p_ready)) {
          tc_fence_after();
          const uint64_t vdesc = smem_desc_sw128(smem_addr(v_ring + ps * C::kVBytes));
#pragma unroll
          for (int kk = 0; kk < C::kKeys / 16; ++kk)
            if (issuer)
              umma_f16_ts(tmem_base + C::kOCol, tmem_base + C::kPCol + ps * 32 + 8 * kk,
                          vdesc + static_cast<uint64_t>(kk * 2), idesc_o, (pi | kk) != 0);
          if (issuer) {
            umma_commit(bar_pfree(ps));
            umma_commit(bar_vempty(ps));
          }
          __syncwarp();
          ++pi;
          idle = 0;
          continue;
        }
        if ((++idle & 63) == 0) {
          const uint64_t now = global_timer_ns();
          if (idle == 64) since = now;
          bool stop = *abort_flag != 0;
          if (!stop && now - since > limit) {
            stop = true;
            *abort_flag = 1;
            if (lane == 0) atomicOr(err, kErrWaitUnpack);
          }
          alive = !__any_sync(0xffffffffu, stop);
        }
      }
      if (issuer) umma_commit(bar_o);  // arrives once every MMA of this CTA has completed
      __syncwarp();
      volatile int no_abort = 0;
      mbar_wait_bounded(bar_o, 0, &no_abort, err, kErrWaitDrain, limit);
    }
  } else if (warp >= 12) {
    // ------------------------------------------------ values -> V^T (fp16)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kConvRegs));
    constexpr int W = D / 64;  // words of a lane's run of dims: 1, 2 or 4
    const int kc = lane & 7;   // positions 8 kc .. 8 kc + 7 of a tile: keys kc, kc + 8, ...
    const int dim0 = (warp - 12) * (D / 4) + (lane >> 3) * (D / 16);
    // keys kc + 8 k lie 8 rows apart, with the same swizzle
    const uint8_t* src = v_raw + (D >= 128 ? (dim0 >> 7) * (C::kKeys * 128) + kc * 128 + ((((dim0 >> 4) & 7) ^ kc) << 4)
                                           : kc * 64 + (((dim0 >> 4) ^ ((kc >> 1) & 3)) << 4)) + (dim0 & 15);
    constexpr int kStep = 8 * (D >= 128 ? 128 : 64);
    for (int i = 0; i < nt; ++i) {
      const int slot = i & 1;
      bool ok = mbar_wait_spin(bar_vraw(slot), (i >> 1) & 1, abort_flag, err, kErrWaitTma, limit);
      if (ok && i >= 2) ok = mbar_wait_spin(bar_vempty(slot), ((i >> 1) - 1) & 1, abort_flag, err, kErrWaitEmpty, limit);
      if (!warp_all(ok)) break;
      uint32_t w[8][W];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint8_t* a = src + slot * C::kRaw + k * kStep;
        if constexpr (W == 4) *reinterpret_cast<uint4*>(w[k]) = *reinterpret_cast<const uint4*>(a);
        else if constexpr (W == 2) *reinterpret_cast<uint2*>(w[k]) = *reinterpret_cast<const uint2*>(a);
        else w[k][0] = *reinterpret_cast<const uint32_t*>(a);
      }
      uint8_t* dst = v_ring + slot * C::kVBytes;
#pragma unroll
      for (int x = 0; x < W; ++x) {
        uint32_t lo[4], hi[4];  // pairs of keys of dims 4x, 4x + 1 and 4x + 2, 4x + 3
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t u0 = w[2 * k][x] ^ 0x80808080u, u1 = w[2 * k + 1][x] ^ 0x80808080u;
          lo[k] = __byte_perm(u0, u1, 0x5140);
          hi[k] = __byte_perm(u0, u1, 0x7362);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int dim = dim0 + 4 * x + y;
          const uint32_t(&z)[4] = y < 2 ? lo : hi;
          uint4 o;
          if (y & 1)
            o = make_uint4(codes_to_half2<1>(z[0]), codes_to_half2<1>(z[1]), codes_to_half2<1>(z[2]), codes_to_half2<1>(z[3]));
          else
            o = make_uint4(codes_to_half2<0>(z[0]), codes_to_half2<0>(z[1]), codes_to_half2<0>(z[2]), codes_to_half2<0>(z[3]));
          *reinterpret_cast<uint4*>(dst + dim * 128 + ((kc ^ (dim & 7)) << 4)) = o;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_vread(slot));
        mbar_arrive(bar_vfull(slot));
      }
    }
  } else if (warp >= 8) {
    // ------------------------------------------------ keys -> K (fp16)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kConvRegs));
    constexpr int J = D / 16;          // 16-byte chunks of a key
    constexpr int kPass = 128 / J;     // keys of a pass of the 128 threads
    constexpr int U = C::kKeys / kPass;
    const int t = threadIdx.x - 256, j = t % J, s0 = t / J, sel = (lane >> 2) & 1;
    bool alive = nt == 0 || warp_all(mbar_wait_spin(bar_q, 0, abort_flag, err, kErrWaitUnpack, limit));  // Q has left the ring
    for (int i = 0; alive && i < nt; ++i) {
      const int slot = i & 1;
      bool ok = mbar_wait_spin(bar_kraw(slot), (i >> 1) & 1, abort_flag, err, kErrWaitTma, limit);
      if (ok && i >= 2) ok = mbar_wait_spin(bar_kempty(slot), ((i >> 1) - 1) & 1, abort_flag, err, kErrWaitEmpty, limit);
      if (!warp_all(ok)) break;
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = s0 + kPass * u;  // key of the tile
        w[u] = *reinterpret_cast<const uint4*>(
            k_raw + slot * C::kRaw + (D >= 128 ? (j >> 3) * (C::kKeys * 128) + s * 128 + (((j & 7) ^ (s & 7)) << 4)
                                               : s * 64 + ((j ^ ((s >> 1) & 3)) << 4)));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = s0 + kPass * u, row = 8 * (s & 7) + (s >> 3);
        uint8_t* dst = k_ring + slot * C::kKBytes + (j >> 2) * (C::kKeys * 128) + row * 128;
        const uint32_t x[4] = {w[u].x ^ 0x80808080u, w[u].y ^ 0x80808080u, w[u].z ^ 0x80808080u, w[u].w ^ 0x80808080u};
        uint4 o[2];
#pragma unroll
        for (int y = 0; y < 2; ++y)
          o[y] = make_uint4(codes_to_half2<0>(x[2 * y]), codes_to_half2<1>(x[2 * y]), codes_to_half2<0>(x[2 * y + 1]),
                            codes_to_half2<1>(x[2 * y + 1]));
        // the two halves in turn, so that 8 lanes meet all banks
        const int c = 2 * (j & 3);
        *reinterpret_cast<uint4*>(dst + (((c + sel) ^ (row & 7)) << 4)) = sel ? o[1] : o[0];
        *reinterpret_cast<uint4*>(dst + (((c + 1 - sel) ^ (row & 7)) << 4)) = sel ? o[0] : o[1];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_kread(slot));
        mbar_arrive(bar_kfull(slot));
      }
    }
  } else {
    // ------------------------------------------------ softmax + epilogue (warps 0-7)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftRegs));
    const int quarter = warp & 3, group = warp >> 2;
    const int row = quarter * 32 + lane, r = r0 + row;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    // ---- Q: raw rows to shared memory, then (thread = row and half of its dims) to TMEM as fp16
    {
      cp_async_wait<0>();
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the 8 softmax warps (nothing has given up yet)
      const uint8_t* mine = q_smem + row * 2 * D;
      float shift = 1.f;
      if constexpr (!std::is_same_v<T, __half>) {
        // bf16: the row's largest element decides the power of two that brings it into fp16
        __nv_bfloat162 top = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll 4
        for (int c = group * (QC / 2); c < (group + 1) * (QC / 2); ++c) {
          const uint4 raw = *reinterpret_cast<const uint4*>(mine + ((c ^ (row & 7)) << 4));
          const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
          for (int e = 0; e < 4; ++e) top = __hmax2(top, __habs2(x[e]));
        }
        row_x[group * C::kRows + row] = fmaxf(__low2float(top), __high2float(top));
        asm volatile("bar.sync 1, 256;" ::: "memory");
        shift = query_shift(fmaxf(row_x[row], row_x[C::kRows + row]));
      }
      const float up = p.scale < 0.f ? -shift : shift;
      if (group == 0) {
        // rows past the last count as it does (their queries are zero, nothing of theirs is stored): a warp with rows
        // that see less than a tile takes the longer way through it
        row_info[row] = make_float2(fabsf(p.scale) / shift,
                                    __int_as_float(keys_seen(p, n, p.causal ? min(r, p.rows - 1) / p.group : 0)));
        row_r[row] = -INFINITY;
      }
#pragma unroll 1
      for (int c = group * (QC / 2); c < (group + 1) * (QC / 2); c += 4) {
        uint32_t w[16];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint8_t* src = mine + (((c + x) ^ (row & 7)) << 4);
          if constexpr (std::is_same_v<T, __half>) {
            const uint4 raw = *reinterpret_cast<const uint4*>(src);
            const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
            w[4 * x] = raw.x ^ flip, w[4 * x + 1] = raw.y ^ flip, w[4 * x + 2] = raw.z ^ flip, w[4 * x + 3] = raw.w ^ flip;
          } else {
            float v[8];
            load8(reinterpret_cast<const T*>(src), v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 y = __fmul2_rn(make_float2(v[2 * e], v[2 * e + 1]), make_float2(up, up));
              w[4 * x + e] = pack_half2_bits(y.x, y.y);
            }
          }
        }
        tmem_st_32x32b_x16(tmem_base + lane_addr + C::kQCol + 4 * c, w);
      }
      tmem_st_wait();
      tc_fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");  // row_info, row_r; row_x may be written again
      if (lane == 0) mbar_arrive(bar_q);
    }
    const float2 info = row_info[row];
    const float factor = info.x;
    const int seen = __float_as_int(info.y);
    const float* ks = p.ks + static_cast<long long>(unit) * (p.capacity / kKvBlock);
    const float* vs = p.vs + static_cast<long long>(unit) * (p.capacity / kKvBlock);
    float m = -INFINITY, l = 0.f;
    bool alive = true;
    // a tile's scales, one to a lane, a turn ahead: keys' (lanes 0-3), values' (4-7), the exponents of these (8-11); zero
    // past the length
    const float* scale_src = (lane < 4 ? ks : vs) + (lane & 3);
    const auto fetch_scale = [&](int i) {
      const int blk = (tile0 + i) * (C::kKeys / kKvBlock);
      const float v = lane < 12 && i < nt && blk + (lane & 3) < nblocks ? __ldg(scale_src + blk) : 0.f;
      return lane < 8 ? v : value_exponent(v);
    };
    float scales = fetch_scale(group);
    for (int i = group; i < nt; i += 2) {
      const int j0 = (tile0 + i) * C::kKeys;
      float ksc[4], vsc[4], ve[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        ksc[q] = __shfl_sync(0xffffffffu, scales, q) * factor;
        vsc[q] = __shfl_sync(0xffffffffu, scales, 4 + q);
        ve[q] = __shfl_sync(0xffffffffu, scales, 8 + q);
      }
      scales = fetch_scale(i + 2);
      if (!warp_all(mbar_wait_spin(bar_sfull(group), (i >> 1) & 1, abort_flag, err, kErrWaitAccum, limit))) {
        alive = false;
        break;
      }
      tc_fence_after();
      uint32_t raw[64];
#pragma unroll
      for (int c = 0; c < 64; c += 16)
        tmem_ld_32x32b_x16(tmem_base + lane_addr + C::kSCol + c, *reinterpret_cast<uint32_t(*)[16]>(&raw[c]));
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_sread);
      // ---- the row's maxima of the tile, of s and of s + e; column c is key 8 (c % 8) + c / 8, whose scale is number
      // (c % 8) / 2.  Keys that the row does not see are left out, whatever their block's scales
      float bmax = -INFINITY, rmax = -INFINITY;
      const int left = seen - j0;
      const bool whole = __all_sync(0xffffffffu, left >= C::kKeys);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float x0 = -INFINITY, x1 = -INFINITY;
        if (whole) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            x0 = fmaxf(x0, __uint_as_float(raw[8 * c + 2 * q]));
            x1 = fmaxf(x1, __uint_as_float(raw[8 * c + 2 * q + 1]));
          }
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            if (16 * q + c < left) x0 = fmaxf(x0, __uint_as_float(raw[8 * c + 2 * q]));
            if (16 * q + 8 + c < left) x1 = fmaxf(x1, __uint_as_float(raw[8 * c + 2 * q + 1]));
          }
        }
        x0 = fmaxf(x0, x1);
        if (x0 > -INFINITY) {
          x0 *= ksc[q];  // the factor is not negative
          bmax = fmaxf(bmax, x0);
          rmax = fmaxf(rmax, x0 + ve[q]);
        }
      }
      if (bmax > m + kAttn8Grow) {
        bmax += kAttn8Margin;
        l *= m == -INFINITY ? 0.f : ex2_approx(m - bmax);
        m = bmax;
      }
      // ---- r as the tile before left it, then this tile's
      if (i > 0 && !warp_all(mbar_wait_spin(bar_r(quarter), (i - 1) & 1, abort_flag, err, kErrWaitAccum, limit))) {
        alive = false;
        break;
      }
      float ref = row_r[row];
      float f = 1.f;
      if (rmax > ref + kAttn8Grow) {
        rmax += kAttn8Margin;
        f = ref == -INFINITY ? 0.f : ex2_approx(ref - rmax);
        ref = rmax;
      }
      if (i >= 1 && __any_sync(0xffffffffu, f != 1.f)) {
        // O holds the earlier tiles: wait for the last of them, rescale this warp's rows
        if (!warp_all(mbar_wait_spin(bar_pfree((i - 1) & 1), ((i - 1) >> 1) & 1, abort_flag, err, kErrWaitAccum, limit))) {
          alive = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t o[32];
          const uint32_t t = tmem_base + lane_addr + C::kOCol + c0;
          tmem_ld_32x32b_x16(t, *reinterpret_cast<uint32_t(*)[16]>(&o[0]));
          tmem_ld_32x32b_x16(t + 16, *reinterpret_cast<uint32_t(*)[16]>(&o[16]));
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
          tmem_st_32x32b_x32(t, o);
        }
        tmem_st_wait();
        tc_fence_before();
      }
      row_r[row] = ref;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_r(quarter));
      // ---- w = p (vs 2^(m - r))
      const float nm = m == -INFINITY ? 0.f : -m;
      const bool plain = whole && vsc[0] + vsc[1] + vsc[2] + vsc[3] <= kMaxFloat;  // false for NaN
      const float half = half_way(m - ref);
      float rv[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) rv[q] = plain ? value_factor(vsc[q], half) : any_value_factor(vsc[q], half);
      if (i >= 2 && !warp_all(mbar_wait_spin(bar_pfree(group), ((i >> 1) - 1) & 1, abort_flag, err, kErrWaitAccum, limit))) {
        alive = false;
        break;
      }
      tc_fence_after();
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t pw[16];
        if (plain) {
          const float2 mm = make_float2(nm, nm);
#pragma unroll
          for (int c = 0; c < 16; ++c) {  // columns 32 hf + 2c, + 1: scale c % 4
            const int q = c & 3;
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(raw[32 * hf + 2 * c]), __uint_as_float(raw[32 * hf + 2 * c + 1])),
                                        make_float2(ksc[q], ksc[q]), mm);
            const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            sum[c & 1] = __fadd2_rn(sum[c & 1], e);
            const float2 w = __fmul2_rn(e, make_float2(rv[q], rv[q]));
            pw[c] = pack_half2_bits(w.x, w.y);
          }
        } else {
          // a row's last keys, or a block with an infinity or NaN: a key that is not seen counts nothing, whatever its
          // block's scales are
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const int q = c & 3, key = 16 * q + 4 * hf + (c >> 2);
            float e[2];
#pragma unroll
            for (int z = 0; z < 2; ++z)
              e[z] = key + 8 * z < left ? ex2_approx(__fmaf_rn(__uint_as_float(raw[32 * hf + 2 * c + z]), ksc[q], nm)) : 0.f;
            sum[0].x += e[0];
            sum[0].y += e[1];
            pw[c] = pack_half2_bits(weigh(e[0], rv[q]), weigh(e[1], rv[q]));
          }
        }
        tmem_st_32x32b_x16(tmem_base + lane_addr + C::kPCol + 32 * group + 16 * hf, pw);
      }
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_pfull(group));
    }
    // ---- epilogue: O 2^(r - m) / l as T, or without the division and with (m, l) for this split, to shared memory (the
    // idle rings).  Where a wait gave up l is NaN
    alive = alive && warp_all(mbar_wait_bounded(bar_o, 0, abort_flag, err, kErrWaitAccum, limit));
    tc_fence_after();
    row_x[group * C::kRows + row] = l;
    row_m[group * C::kRows + row] = m;
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_l(quarter));
    alive = warp_all(mbar_wait_spin(bar_l(quarter), 0, abort_flag, err, kErrWaitAccum, limit)) && alive;
    {
      const float m0 = row_m[row], m1 = row_m[C::kRows + row];
      m = fmaxf(m0, m1);
      l = (m0 == -INFINITY ? 0.f : row_x[row] * ex2_approx(m0 - m)) +
          (m1 == -INFINITY ? 0.f : row_x[C::kRows + row] * ex2_approx(m1 - m));
    }
    if (!alive) l = __uint_as_float(0x7fc00000u);
    const bool part = p.splits > 1;
    const float back = half_way(row_r[row] - m);  // half of the way from r to m
    const float f = part ? back : back / l;
    if (part && group == 0 && r < p.rows)
      p.part_ml[(static_cast<long long>(unit) * p.splits + split) * p.rows + r] = make_float2(m, l);
#pragma unroll 1
    for (int c0 = group * (D / 2); c0 < (group + 1) * (D / 2); c0 += 16) {
      uint32_t o[16];
      if (nt > 0) {
        tmem_ld_32x32b_x16(tmem_base + lane_addr + C::kOCol + c0, o);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int c = 0; c < 16; ++c) o[c] = 0u;
      }
      float v[2][8];
#pragma unroll
      for (int c = 0; c < 16; ++c) v[c >> 3][c & 7] = l == 0.f ? 0.f : __uint_as_float(o[c]) * back * f;
      if (part) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<float4*>(base + row * 4 * D + (((c0 / 4 + c) ^ (row & 7)) << 4)) =
              make_float4(v[c >> 1][4 * (c & 1)], v[c >> 1][4 * (c & 1) + 1], v[c >> 1][4 * (c & 1) + 2], v[c >> 1][4 * (c & 1) + 3]);
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c)
          store8(reinterpret_cast<T*>(base + row * 2 * D + (((c0 / 8 + c) ^ (row & 7)) << 4)), v[c]);
      }
    }
    fence_proxy_async_smem();
  }
  // every MMA has completed (the issuer waited for bar_o) before TMEM is freed
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
  const int rows = min(C::kRows, p.rows - r0);
  if (p.splits > 1) {
    // the rows lie in the workspace as in shared memory (chunk c of row r at c ^ (r & 7)): one copy
    if (threadIdx.x == 0) {
      bulk_store(p.part_o + ((static_cast<long long>(unit) * p.splits + split) * p.rows + r0) * D, smem_addr(base),
                 static_cast<uint32_t>(rows) * 4 * D);
      bulk_commit_group();
      bulk_wait_group0();
    }
  } else {
    for (int i = warp; i < rows; i += C::kThreads / 32)
      if (lane < QC)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + out_row(p, b, h, r0 + i) * D + lane * 8) =
            *reinterpret_cast<const uint4*>(base + i * 2 * D + ((lane ^ (i & 7)) << 4));
  }
}

// out[row] = sum_s O_s 2^(m_s - m) / sum_s l_s 2^(m_s - m): one CTA of THREADS
// per row, a thread with one 16-byte chunk of every (4 THREADS / D)-th part
// (chunk c of row r lies at c ^ (r & 7)).  m first, from all parts' m_s, so that
// the parts' loads do not wait for one another.  128 threads for up to 32 parts;
// 512 for more (8 rows of width 256, 64 parts: 21.1 us with the attention in one
// pass of 128 threads, 10.4 so).
template <typename T, int D, int THREADS>
__global__ void __launch_bounds__(THREADS) attn8_join_kernel(const __grid_constant__ Attn8Params p) {
  constexpr int NC = D / 4, G = THREADS / NC;
  __shared__ float4 red[G][NC];
  __shared__ float red_l[G];
  pdl_launch_dependents();
  pdl_wait();
  const int c = threadIdx.x % NC, g = threadIdx.x / NC;
  const int r = blockIdx.x, unit = blockIdx.y;
  const long long first = static_cast<long long>(unit) * p.splits * p.rows + r;
  const float2* part_ml = p.part_ml + first;
  float m = -INFINITY;
  for (int s = threadIdx.x & 31; s < p.splits; s += 32) {
    const float2 ml = part_ml[static_cast<long long>(s) * p.rows];
    if (ml.y != 0.f) m = fmaxf(m, ml.x);  // l = 0: saw nothing (a NaN stays)
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int s = g; s < p.splits; s += G) {
    const float2 ml = part_ml[static_cast<long long>(s) * p.rows];
    const float4 v = *reinterpret_cast<const float4*>(p.part_o + (first + static_cast<long long>(s) * p.rows) * D +
                                                      (c ^ (r & 7)) * 4);
    const bool saw = ml.y != 0.f;
    const float f = ex2_approx(ml.x - m);
    sum = saw ? fmaf(ml.y, f, sum) : sum;
    acc.x = saw ? fmaf(v.x, f, acc.x) : acc.x;
    acc.y = saw ? fmaf(v.y, f, acc.y) : acc.y;
    acc.z = saw ? fmaf(v.z, f, acc.z) : acc.z;
    acc.w = saw ? fmaf(v.w, f, acc.w) : acc.w;
  }
  red[g][c] = acc;
  if (c == 0) red_l[g] = sum;
  __syncthreads();
  if (g > 0) return;
  float4 x = red[0][c];
  float total = red_l[0];
#pragma unroll
  for (int w = 1; w < G; ++w) {
    const float4 v = red[w][c];
    x = make_float4(x.x + v.x, x.y + v.y, x.z + v.z, x.w + v.w);
    total += red_l[w];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int b = unit / p.heads, h = unit - b * p.heads;
  store4(static_cast<T*>(p.out) + out_row(p, b, h, r) * D + 4 * c, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
}

}  // namespace w4a4
