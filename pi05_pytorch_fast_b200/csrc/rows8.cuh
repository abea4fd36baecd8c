// Rows in signed 8 bits with one fp32 scale each: the input side of the
// int8 matrix product (gemm8.cuh).
//
// For a row v of h values: scale = fl(amax|v| / 127), codes = rint(v / scale).
// The row kernels differ in where v comes from:
//   kRowQuant  v = x
//   kRowGeglu  v = gelu_tanh(x) * up
//   kRowNorm   s = x + gate * delta;  v = s rsqrt(mean s^2 + eps) gain + shift
// (delta, gate and shift optional; gain, shift and gate one row for all, or one
// for each observation of rows_per_batch rows).  All arithmetic is fp32; s is
// rounded once, to the stream's type, where it is stored as `total`, and the
// norm is taken of the unrounded s.  A row whose scale is zero has zero codes;
// a row with an infinity or NaN gets a non-finite scale and zero codes, so that
// its values (code x scale) are NaN and the fault stays visible.
//
// Bound: HBM (a norm row of bf16 moves 7 bytes per element at about 30
// instructions).  A row is read once and stays in registers through both
// reductions, one CTA of h / (8 VPT) threads per row.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace w4a4 {

enum RowOp : int { kRowQuant = 0, kRowGeglu = 1, kRowNorm = 2 };

// Longest rows held in registers: 8-element vectors (aligned rows), single
// elements (any row); longer ones are read again for each pass.
constexpr int kRow8MaxVec = 32768;
constexpr int kRow8MaxScalar = 16384;

constexpr float kInv127 = 1.0f / 127.0f;

struct Row8Params {
  const void* x;      // [rows, h], row stride ldx
  const void* x2;     // delta or up, row stride ld2 (NULL: none)
  const void* gate;   // multiplies delta (NULL: 1)
  const float* gain;  // kRowNorm
  const float* shift; // NULL: 0
  void* total;        // x + gate delta, contiguous rows (NULL: not stored)
  int8_t* codes;      // row stride ldc
  float* scale;       // [rows]
  long long ldx, ld2, ldc;
  long long gate_stride, gain_stride, shift_stride;  // per observation (0: shared)
  long long rows;
  int rows_per_batch;
  int h;
  float eps;
};

// 8 consecutive elements <-> fp32 (16-byte aligned rows).
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  uint4 raw;
  __half2* h = reinterpret_cast<__half2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint4 raw;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }

// W = 8 or 1 elements.
template <int W, typename T>
__device__ __forceinline__ void load_w(const T* p, float (&v)[W]) {
  if constexpr (W == 8) load8(p, v);
  else v[0] = to_float(*p);
}
template <int W, typename T>
__device__ __forceinline__ void store_w(T* p, const float (&v)[W]) {
  if constexpr (W == 8) store8(p, v);
  else *p = from_float<T>(v[0]);
}

// gelu(x) = x / (1 + exp(-2 u)), u = sqrt(2/pi) (x + 0.044715 x^3): the tanh
// form 0.5 x (1 + tanh u) with 1 + tanh u = 2 / (1 + exp(-2 u)), which does not
// cancel for negative u.
__device__ __forceinline__ float gelu_tanh_f32(float x) {
  const float u2 = 1.5957691216057308f * fmaf(0.044715f * x * x, x, x);
  return __fdividef(x, 1.0f + __expf(-u2));
}

// How codes of a value are formed from a row's (block's) scale: a multiply by
// the reciprocal, which can move a value within an ulp of a rounding tie to
// the other side, or, for scales whose reciprocal would overflow, a division.
struct Coder {
  float mul, div;
  __device__ __forceinline__ explicit Coder(float scale) {
    const bool finite = scale <= 3.4028234e38f;  // false for NaN
    const bool tiny = scale < 7.8886091e-31f;    // 2^-100
    mul = finite && !tiny ? __frcp_rn(scale) : 0.f;
    div = finite && tiny && scale > 0.f ? scale : 0.f;
  }
  __device__ __forceinline__ int operator()(float v) const {
    float t = v * mul;
    if (div != 0.f) t = __fdiv_rn(v, div);
    // a NaN (a non-finite row: inf * 0) becomes code 0
    return t == t ? __float2int_rn(fminf(fmaxf(t, -127.f), 127.f)) : 0;
  }
};

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
template <int W>
__device__ __forceinline__ void store_codes(int8_t* p, const float (&v)[W], const Coder& code) {
  if constexpr (W == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack4(code(v[0]), code(v[1]), code(v[2]), code(v[3])),
                                              pack4(code(v[4]), code(v[5]), code(v[6]), code(v[7])));
  } else {
    *p = static_cast<int8_t>(code(v[0]));
  }
}

// |v| as an unsigned key: ordered like the value, infinity above every finite
// value and NaN above infinity, so a maximum of keys keeps a NaN.
__device__ __forceinline__ uint32_t abs_key(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Reductions over a CTA of whole warps; `red` has 32 words; every thread gets
// the result.  Two calls in a row need different buffers.
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0u;
  return __reduce_max_sync(0xffffffffu, v);
}

// x (and delta / up) at element e of a row -> the value before the norm.
template <int OP, int W, typename T>
__device__ __forceinline__ void row8_load(const Row8Params& p, const T* x, const T* x2, const T* gate, int e,
                                          float (&v)[W]) {
  load_w<W>(x + e, v);
  if constexpr (OP == kRowGeglu) {
    float u[W];
    load_w<W>(x2 + e, u);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = gelu_tanh_f32(v[i]) * u[i];
  } else if constexpr (OP == kRowNorm) {
    if (x2) {
      float d[W];
      load_w<W>(x2 + e, d);
      if (gate) {
        float g[W];
        load_w<W>(gate + e, g);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = fmaf(g[i], d[i], v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] += d[i];
      }
    }
  }
}

template <int W>
__device__ __forceinline__ void row8_norm(const float* gain, const float* shift, int e, float rstd, float (&v)[W]) {
  float g[W];
  load_w<W>(gain + e, g);
  if (shift) {
    float b[W];
    load_w<W>(shift + e, b);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = fmaf(v[i] * rstd, g[i], b[i]);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = v[i] * rstd * g[i];
  }
}

// One row per CTA, held in registers: thread t has the W-element groups
// t, t + blockDim, ... (VPT of them).
template <typename T, int OP, int W, int VPT>
__global__ void __launch_bounds__(1024) row8_kernel(const __grid_constant__ Row8Params p) {
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  pdl_launch_dependents();
  pdl_wait();
  const long long row = blockIdx.x;
  const long long obs = row / p.rows_per_batch;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* x2 = p.x2 ? static_cast<const T*>(p.x2) + row * p.ld2 : nullptr;
  const T* gate = p.gate ? static_cast<const T*>(p.gate) + obs * p.gate_stride : nullptr;
  const int groups = (p.h + W - 1) / W;  // W = 8: h is a multiple of 8
  float v[VPT][W];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int g = threadIdx.x + j * blockDim.x;
    if (g < groups) {
      row8_load<OP, W, T>(p, x, x2, gate, g * W, v[j]);
      if constexpr (OP == kRowNorm) {
        if (p.total) store_w<W>(static_cast<T*>(p.total) + row * p.h + g * W, v[j]);
#pragma unroll
        for (int i = 0; i < W; ++i) ss = fmaf(v[j][i], v[j][i], ss);
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) v[j][i] = 0.f;
    }
  }
  if constexpr (OP == kRowNorm) {
    const float rstd = rsqrtf(block_sum(ss, red_sum) / static_cast<float>(p.h) + p.eps);
    const float* gain = p.gain + obs * p.gain_stride;
    const float* shift = p.shift ? p.shift + obs * p.shift_stride : nullptr;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int g = threadIdx.x + j * blockDim.x;
      if (g < groups) row8_norm<W>(gain, shift, g * W, rstd, v[j]);
    }
  }
  uint32_t key = 0;
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int i = 0; i < W; ++i) key = max(key, abs_key(v[j][i]));
  const float scale = __uint_as_float(block_max(key, red_max)) * kInv127;
  const Coder code(scale);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int g = threadIdx.x + j * blockDim.x;
    if (g < groups) store_codes<W>(p.codes + row * p.ldc + g * W, v[j], code);
  }
  if (threadIdx.x == 0) p.scale[row] = scale;
}

// Rows too long for registers: each pass reads the row again (from L2).
template <typename T, int OP>
__global__ void __launch_bounds__(1024) row8_long_kernel(const __grid_constant__ Row8Params p) {
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  pdl_launch_dependents();
  pdl_wait();
  const long long row = blockIdx.x;
  const long long obs = row / p.rows_per_batch;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* x2 = p.x2 ? static_cast<const T*>(p.x2) + row * p.ld2 : nullptr;
  const T* gate = p.gate ? static_cast<const T*>(p.gate) + obs * p.gate_stride : nullptr;
  const float* gain = nullptr;
  const float* shift = nullptr;
  float rstd = 0.f;
  if constexpr (OP == kRowNorm) {
    gain = p.gain + obs * p.gain_stride;
    shift = p.shift ? p.shift + obs * p.shift_stride : nullptr;
    float ss = 0.f;
    for (int e = threadIdx.x; e < p.h; e += blockDim.x) {
      float v[1];
      row8_load<OP, 1, T>(p, x, x2, gate, e, v);
      if (p.total) store_w<1>(static_cast<T*>(p.total) + row * p.h + e, v);
      ss = fmaf(v[0], v[0], ss);
    }
    rstd = rsqrtf(block_sum(ss, red_sum) / static_cast<float>(p.h) + p.eps);
  }
  uint32_t key = 0;
  for (int e = threadIdx.x; e < p.h; e += blockDim.x) {
    float v[1];
    row8_load<OP, 1, T>(p, x, x2, gate, e, v);
    if constexpr (OP == kRowNorm) row8_norm<1>(gain, shift, e, rstd, v);
    key = max(key, abs_key(v[0]));
  }
  const float scale = __uint_as_float(block_max(key, red_max)) * kInv127;
  const Coder code(scale);
  for (int e = threadIdx.x; e < p.h; e += blockDim.x) {
    float v[1];
    row8_load<OP, 1, T>(p, x, x2, gate, e, v);
    if constexpr (OP == kRowNorm) row8_norm<1>(gain, shift, e, rstd, v);
    store_codes<1>(p.codes + row * p.ldc + e, v, code);
  }
  if (threadIdx.x == 0) p.scale[row] = scale;
}

// out[r, :] = codes[r, :] * scale[r], rounded once; grid (column groups of
// 256 x W, rows).
template <typename T, int W>
__global__ void __launch_bounds__(256) dequant8_kernel(const int8_t* __restrict__ codes, long long ldc,
                                                       const float* __restrict__ scale, T* __restrict__ out,
                                                       long long rows, int h) {
  pdl_launch_dependents();
  pdl_wait();
  const int e = (blockIdx.x * 256 + threadIdx.x) * W;
  if (e >= h) return;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    const float s = scale[row];
    float v[W];
    if constexpr (W == 8) {
      const uint2 raw = *reinterpret_cast<const uint2*>(codes + row * ldc + e);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? raw.x : raw.y) >> (8 * (i & 3)))) * s;
    } else {
      v[0] = static_cast<float>(codes[row * ldc + e]) * s;
    }
    store_w<W>(out + row * h + e, v);
  }
}

}  // namespace w4a4
