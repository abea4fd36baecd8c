// Attention of new queries over the 8-bit key/value cache (kv8.cuh).
//
// Query token t of T, head g of the H / heads that share key/value head h:
//   S[j] = scale * (q . kc[j]) * ks[j / 16],  P = softmax(S),  O = sum_j P[j] vs[j / 16] vc[j]
// over the keys j < lengths[b] (causal: j < lengths[b] - T + t + 1, the
// queries being the last T tokens of the cache).  A query that sees no key
// gives zeros.
#pragma once

#include "kv8.cuh"

namespace w4a4 {

struct Attn8Params {
  const void* q;  // [batch, tokens, q_heads, width]
  void* out;      // contiguous
  const int8_t* k;
  const int8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* lengths;
  long long qb, qt, qh;    // query strides (elements)
  long long cb, ct, ch;    // cache strides
  int batch, tokens, q_heads, heads, width, capacity;
  int causal;
  float scale;
};

// One warp per query row, one key at a time: right for every case.
template <typename T>
__global__ void __launch_bounds__(128) attn8_simple_kernel(const __grid_constant__ Attn8Params p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<long long>(p.batch) * p.tokens * p.q_heads) return;
  const int qh = static_cast<int>(row % p.q_heads);
  const int t = static_cast<int>(row / p.q_heads % p.tokens);
  const int b = static_cast<int>(row / p.q_heads / p.tokens);
  const int h = qh / (p.q_heads / p.heads);
  const T* q = static_cast<const T*>(p.q) + b * p.qb + t * p.qt + qh * p.qh;
  const int per = p.width / 32;  // 2, 4, 6 or 8 elements per lane
  float qv[8], acc[8] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) qv[i] = i < per ? to_float(q[lane + 32 * i]) : 0.f;
  int keys = min(max(p.lengths[b], 0), p.capacity);
  if (p.causal) keys = min(keys, keys - p.tokens + t + 1);
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < keys; ++j) {
    const int8_t* k = p.k + b * p.cb + j * p.ct + h * p.ch;
    const int8_t* v = p.v + b * p.cb + j * p.ct + h * p.ch;
    const long long blk = (static_cast<long long>(b) * p.heads + h) * (p.capacity / kKvBlock) + j / kKvBlock;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < per) s = fmaf(qv[i], static_cast<float>(k[lane + 32 * i]), s);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= p.scale * p.ks[blk];
    const float mn = fmaxf(m, s);
    const float a = __expf(m - mn), e = __expf(s - mn);
    l = l * a + e;
    m = mn;
    const float w = e * p.vs[blk];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < per) acc[i] = fmaf(w, static_cast<float>(v[lane + 32 * i]), acc[i] * a);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* out = static_cast<T*>(p.out) + row * p.width;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < per) out[lane + 32 * i] = from_float<T>(acc[i] * inv);
}

}  // namespace w4a4
