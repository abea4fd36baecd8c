// The 8-bit key/value cache: int8 codes [batch, capacity, heads, width] for
// keys and values each, and one fp32 scale for each block of 16 consecutive
// tokens and head, [batch, heads, capacity / 16].  A value is code x scale.
//
// Appending (kv8_append_kernel).  Observation b's valid new tokens go, in
// order and without gaps, to the slots from start[b] on.  Per block that
// receives tokens and per head, with x the new values in it:
//   scale' = max(scale if the block keeps earlier tokens, amax|x| * fl(1 / 127))
//   new codes = rint(x / scale'),  kept codes = rint(code * (scale / scale'))
// so a block that is filled over several calls is rounded again only when its
// scale grows, and one whose scale does not grow keeps its codes: writing the
// same tokens to the same slots again changes nothing.  A block that is begun
// anew (its first slot is >= start[b]) forgets its old scale.  An infinity or
// NaN among x makes the block's scale non-finite and its codes zero.
//
// Bound: HBM (2 bytes read and 1 written per value), or for short appends the
// chain of loads flags -> tokens -> codes.  One CTA per block and head for keys
// and values together, a thread to 8 elements of one slot of each, which stay in
// registers between the maximum and the rounding.  Every warp counts the valid
// tokens for itself, 1,024 flags at a time, and finds those of its own slots: no
// earlier kernel, no barrier, no list in memory.  Measured: 8 x 776 tokens of
// width 256 4.7 us, with flags 7.4; 8 x 1 token 2.5 us.
#pragma once

#include "rows8.cuh"

namespace w4a4 {

constexpr int kKvBlock = 16;  // tokens that share a scale

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

// The token whose rank among an observation's valid tokens is r0 + (the calling
// thread's slot), or -1, and the number of valid tokens.  A warp has 256 / width
// slots, the first of them `slot0`, and calls as a whole.
__device__ __forceinline__ int find_token(const uint8_t* valid, int tokens, long long r0, int slot0, int slot, int width,
                                          int& count) {
  if (!valid) {
    const long long r = r0 + slot;
    count = tokens;
    return r >= 0 && r < tokens ? static_cast<int>(r) : -1;
  }
  // words of four flags from the last address before the row that is a multiple of 4 on; the row's ends go by bytes
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(valid) & 3);
  const int lane = threadIdx.x & 31;
  int found = -1;
  count = 0;
  for (int t0 = -lead; t0 < tokens; t0 += 1024) {
    const int t = t0 + 32 * lane;
    uint32_t f = 0;  // 32 flags
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int u = t + 4 * i;
      uint32_t w = 0;
      if (u >= 0 && u + 4 <= tokens) {
        w = __vcmpne4(*reinterpret_cast<const uint32_t*>(valid + u), 0u) & 0x01010101u;
      } else if (u < tokens) {
        for (int j = max(0, -u); j < 4 && u + j < tokens; ++j) w |= static_cast<uint32_t>(valid[u + j] != 0) << (8 * j);
      }
      f |= (w * 0x01020408u >> 24) << (4 * i);  // the four bytes' lowest bits, side by side
    }
    const int n = __popc(f);
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const int all = __shfl_sync(0xffffffffu, incl, 31);
    for (int k = 0; k < 256 / width; ++k) {
      const long long want = r0 + slot0 + k - count;  // its rank among these 1,024
      if (want < 0 || want >= all) continue;
      const int left = static_cast<int>(want) - (incl - n);
      int token = -1;
      if (left >= 0 && left < n) {
        uint32_t rest = f;
        for (int i = 0; i < left; ++i) rest &= rest - 1;
        token = t + __ffs(rest) - 1;
      }
      token = __reduce_max_sync(0xffffffffu, token);
      if (slot == slot0 + k) found = token;
    }
    count += all;
  }
  return found;
}

// grid (blocks that a run of `tokens` slots can touch, batch * heads), 2 x width
// threads.  VEC: the new values' rows begin at multiples of 16 bytes.
template <typename T, bool VEC>
__global__ void __launch_bounds__(512, 3) kv8_append_kernel(const __grid_constant__ Kv8Params p) {
  __shared__ uint32_t red[2][16];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y / p.heads, h = blockIdx.y - b * p.heads;
  const int per = p.width / 8, slot = threadIdx.x / per, e = (threadIdx.x % per) * 8;
  const int start = p.start[b];
  const bool bad = start < 0 || start > p.capacity;
  const int first = bad ? 0 : start / kKvBlock + static_cast<int>(blockIdx.x);
  const long long s0 = static_cast<long long>(first) * kKvBlock;  // the block's first slot
  int count;
  const int token = find_token(p.valid ? p.valid + b * p.valid_stride : nullptr, p.tokens, s0 - start,
                               (threadIdx.x & ~31) / per, slot, p.width, count);
  const long long end = static_cast<long long>(start) + count;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
    p.lengths[b] = bad ? max(0, min(start, p.capacity)) : static_cast<int>(min(end, static_cast<long long>(p.capacity)));
    if (bad || end > p.capacity) atomicOr(&g_w4a4_device_error, kErrCacheFull);
  }
  if (bad || s0 >= end || s0 >= p.capacity) return;
  const int kept = start > s0 ? static_cast<int>(start - s0) : 0;  // earlier tokens that stay
  const bool keeps = slot < kept;
  const long long at = b * p.cb + (s0 + slot) * p.ct + h * p.ch + e;
  const long long at_scale = (static_cast<long long>(b) * p.heads + h) * (p.capacity / kKvBlock) + first;
  float v[2][8] = {}, was[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    was[i] = kept ? p.scale[i][at_scale] : 0.f;
    if (token >= 0) {
      const T* x = static_cast<const T*>(p.x[i]) + b * p.xb[i] + h * p.xh[i] + token * p.xt[i] + e;
      if constexpr (VEC) {
        load8(x, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = to_float(x[j]);
      }
    } else if (keeps) {
      const uint2 raw = *reinterpret_cast<const uint2*>(p.codes[i] + at);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[i][j] = static_cast<float>(static_cast<int8_t>((j < 4 ? raw.x : raw.y) >> (8 * (j & 3))));
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t key = 0;
    if (token >= 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) key = max(key, abs_key(v[i][j]));
    }
    key = __reduce_max_sync(0xffffffffu, key);
    if ((threadIdx.x & 31) == 0) red[i][threadIdx.x >> 5] = key;
  }
  __syncthreads();  // also: every thread has read the old scales
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int lane = threadIdx.x & 31;
    const uint32_t key = __reduce_max_sync(0xffffffffu, lane < static_cast<int>(blockDim.x >> 5) ? red[i][lane] : 0u);
    // keeps a NaN of either side
    const float now = __uint_as_float(max(abs_key(was[i]), abs_key(__uint_as_float(key) * kInv127)));
    if (threadIdx.x == 0) p.scale[i][at_scale] = now;
    if (token >= 0) {
      store_codes(p.codes[i] + at, v[i], Coder(now));
    } else if (keeps && was[i] != now) {
      // in steps of the new scale, as if the scale were one
      const float ratio = now > 0.f && now <= 3.4028234e38f ? __fdiv_rn(was[i], now) : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= ratio;
      store_codes(p.codes[i] + at, v[i], Coder(1.f));
    }
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

// The values the cache stands for, zero from lengths[b] on.  grid (blocks of 16
// tokens, batch * heads, 2), a thread to 16 codes: `width` threads.  Bound: HBM;
// 8 x 832 slots of width 256 3.7 us (10 MB).
template <typename T>
__global__ void __launch_bounds__(256) kv8_values_kernel(const __grid_constant__ Kv8ValuesParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y / p.heads, h = blockIdx.y - b * p.heads, which = blockIdx.z;
  const int token = blockIdx.x * kKvBlock + threadIdx.x / (p.width / 16), e = (threadIdx.x % (p.width / 16)) * 16;
  const float s = p.scale[which][static_cast<long long>(blockIdx.y) * (p.capacity / kKvBlock) + blockIdx.x];
  T* out = static_cast<T*>(p.out[which]) + ((static_cast<long long>(b) * p.capacity + token) * p.heads + h) * p.width + e;
  uint4 raw = {};
  const bool filled = token < p.lengths[b];
  if (filled) raw = *reinterpret_cast<const uint4*>(p.codes[which] + b * p.cb + token * p.ct + h * p.ch + e);
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = filled ? static_cast<float>(static_cast<int8_t>(w[2 * half + (j >> 2)] >> (8 * (j & 3)))) * s : 0.f;
    store8(out + 8 * half, v);
  }
}

}  // namespace w4a4
