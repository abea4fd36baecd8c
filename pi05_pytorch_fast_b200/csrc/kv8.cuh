// The 8-bit key/value cache: int8 codes [batch, capacity, heads, width] for
// keys and values each, and one fp32 scale for each block of 16 consecutive
// tokens and head, [batch, heads, capacity / 16].  A value is code x scale.
//
// Appending (kv8_append_kernel).  Observation b's valid new tokens go, in
// order and without gaps, to the slots from start[b] on.  Per block that
// receives tokens and per head, with x the new values in it:
//   scale' = max(scale if the block keeps earlier tokens, fl(amax|x| / 127))
//   new codes = rint(x / scale'),  kept codes = rint(code * (scale / scale'))
// so a block that is filled over several calls is rounded again only when its
// scale grows, and one whose scale does not grow keeps its codes: writing the
// same tokens to the same slots again changes nothing.  A block that is begun
// anew (its first slot is >= start[b]) forgets its old scale.  An infinity or
// NaN among x makes the block's scale non-finite and its codes zero.
//
// Bound: HBM, or the launch for a few tokens (2 bytes read and 1 written per
// value).  One CTA per block, head and {keys, values}.
#pragma once

#include "rows8.cuh"

namespace w4a4 {

constexpr int kKvBlock = 16;  // tokens that share a scale
constexpr int kKvThreads = 256;

struct Kv8Params {
  int8_t* codes[2];        // keys, values
  float* scale[2];         // contiguous [batch, heads, capacity / 16]
  const void* x[2];        // new keys, values [batch, tokens, heads, width]
  const int32_t* start;    // [batch]
  const uint8_t* valid;    // [batch, tokens], or NULL: all
  int32_t* lengths;        // [batch] out
  long long cb, ct, ch;    // cache strides (elements) of batch, token, head
  long long xb[2], xt[2], xh[2];
  long long valid_stride;
  int batch, tokens, heads, width, capacity;
};

// Source tokens of ranks [r0, r0 + 16) among the valid tokens of one
// observation, into src[16] (-1: none), and the number of valid tokens.  All
// 256 threads; `red` has 8 words.
__device__ __forceinline__ int find_valid_tokens(const uint8_t* valid, int tokens, long long r0, int* src, int* red) {
  if (threadIdx.x < kKvBlock) {
    const long long r = r0 + threadIdx.x;
    src[threadIdx.x] = !valid && r >= 0 && r < tokens ? static_cast<int>(r) : -1;
  }
  __syncthreads();
  if (!valid) return tokens;
  int base = 0;
  for (int t0 = 0; t0 < tokens; t0 += 4 * kKvThreads) {
    const int t = t0 + 4 * threadIdx.x;
    int f[4], n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = t + i < tokens && valid[t + i] != 0;
      n += f[i];
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if ((threadIdx.x & 31) >= o) incl += u;
    }
    if ((threadIdx.x & 31) == 31) red[threadIdx.x >> 5] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kKvThreads / 32; ++w) {
      if (w < static_cast<int>(threadIdx.x >> 5)) before += red[w];
      all += red[w];
    }
    long long r = static_cast<long long>(base) + before + incl - n - r0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (f[i] && r >= 0 && r < kKvBlock) src[r] = t + i;
      r += f[i];
    }
    base += all;
    __syncthreads();
  }
  return base;
}

// grid (ceil((tokens + 14) / 16) + ..., batch * heads, 2); W = 8 or 1 elements.
template <typename T, int W>
__global__ void __launch_bounds__(kKvThreads) kv8_append_kernel(const __grid_constant__ Kv8Params p) {
  __shared__ int src[kKvBlock];
  __shared__ int red[kKvThreads / 32];
  __shared__ uint32_t red_max[32];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y / p.heads, h = blockIdx.y - b * p.heads, which = blockIdx.z;
  const int start = p.start[b];
  const bool bad = start < 0 || start > p.capacity;
  const int first = bad ? 0 : start / kKvBlock + static_cast<int>(blockIdx.x);
  const long long s0 = static_cast<long long>(first) * kKvBlock;  // the block's first slot
  const int count = find_valid_tokens(p.valid ? p.valid + b * p.valid_stride : nullptr, p.tokens, s0 - start, src, red);
  const long long end = static_cast<long long>(start) + count;
  if (blockIdx.x == 0 && h == 0 && which == 0 && threadIdx.x == 0) {
    p.lengths[b] = bad ? max(0, min(start, p.capacity)) : static_cast<int>(min(end, static_cast<long long>(p.capacity)));
    if (bad || end > p.capacity) atomicOr(&g_w4a4_device_error, kErrCacheFull);
  }
  if (bad || s0 >= end || s0 >= p.capacity) return;
  const T* x = static_cast<const T*>(p.x[which]) + b * p.xb[which] + h * p.xh[which];
  int8_t* codes = p.codes[which] + b * p.cb + s0 * p.ct + h * p.ch;
  float* scale = p.scale[which] + (static_cast<long long>(b) * p.heads + h) * (p.capacity / kKvBlock) + first;
  const int groups = p.width / W, total = kKvBlock * groups;
  uint32_t key = 0;
  for (int i = threadIdx.x; i < total; i += kKvThreads) {
    const int t = i / groups, e = (i - t * groups) * W;
    if (src[t] >= 0) {
      float v[W];
      load_w<W>(x + src[t] * p.xt[which] + e, v);
#pragma unroll
      for (int j = 0; j < W; ++j) key = max(key, abs_key(v[j]));
    }
  }
  const float fresh = __uint_as_float(block_max(key, red_max)) * kInv127;
  const int kept = start > s0 ? static_cast<int>(start - s0) : 0;  // earlier tokens that stay
  const float was = kept ? *scale : 0.f;
  // keeps a NaN of either side
  const float now = __uint_as_float(max(abs_key(was), abs_key(fresh)));
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *scale = now;
  const float ratio = now > 0.f ? __fdiv_rn(was, now) : 0.f;
  const bool usable = now > 0.f && now <= 3.4028234e38f;
  for (int i = threadIdx.x; i < total; i += kKvThreads) {
    const int t = i / groups, e = (i - t * groups) * W;
    int8_t* dst = codes + t * p.ct + e;
    int c[W];
    if (t < kept) {
      if (ratio == 1.f) continue;
#pragma unroll
      for (int j = 0; j < W; ++j) c[j] = usable ? __float2int_rn(static_cast<float>(dst[j]) * ratio) : 0;
    } else if (src[t] >= 0) {
      float v[W];
      load_w<W>(x + src[t] * p.xt[which] + e, v);
#pragma unroll
      for (int j = 0; j < W; ++j)
        c[j] = usable ? __float2int_rn(fminf(fmaxf(__fdiv_rn(v[j], now), -127.f), 127.f)) : 0;
    } else {
      continue;
    }
    if constexpr (W == 8)
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
    else
      dst[0] = static_cast<int8_t>(c[0]);
  }
}

struct Kv8ValuesParams {
  const int8_t* codes[2];
  const float* scale[2];
  void* out[2];            // [batch, capacity, heads, width] contiguous
  const int32_t* lengths;
  long long cb, ct, ch;
  int batch, heads, width, capacity;
};

// The values the cache stands for, zero from lengths[b] on.  grid (groups of
// 256 x 8 values of one token block of all heads..., batch, 2).
template <typename T>
__global__ void __launch_bounds__(256) kv8_values_kernel(const __grid_constant__ Kv8ValuesParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y, which = blockIdx.z;
  const int per_head = p.width / 8, per_token = p.heads * per_head;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long token = i / per_token;
  if (token >= p.capacity) return;
  const int rem = static_cast<int>(i - token * per_token);
  const int h = rem / per_head, e = (rem - h * per_head) * 8;
  float v[8] = {};
  if (token < p.lengths[b]) {
    const float s = p.scale[which][(static_cast<long long>(b) * p.heads + h) * (p.capacity / kKvBlock) + token / kKvBlock];
    const uint2 raw = *reinterpret_cast<const uint2*>(p.codes[which] + b * p.cb + token * p.ct + h * p.ch + e);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = static_cast<float>(static_cast<int8_t>((j < 4 ? raw.x : raw.y) >> (8 * (j & 3)))) * s;
  }
  store8(static_cast<T*>(p.out[which]) + ((static_cast<long long>(b) * p.capacity + token) * p.heads + h) * p.width + e, v);
}

}  // namespace w4a4
