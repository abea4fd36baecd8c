// Rows in signed 8 bits with one fp32 scale each: the input side of the
// int8 matrix product (gemm8.cuh).
//
// For a row v of h values, in fp32: scale = amax|v| * fl(1 / 127), codes =
// rint(v / scale), the quotient rounded as a division does and ties to even.
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
// Bound: HBM.  A row is read once and stays in registers through both
// reductions, one CTA of h / (8 VPT) threads to a row; a CTA takes several rows
// in turn, and asks for the next one's vectors before it reduces this one, so
// that loads are under way all the time.  The arithmetic is two lanes wide
// (f32x2), as at the memory's rate there are about 25 issue slots for an element
// of the GeGLU.  Measured: norm of 49,664 x 2,048 with residual 118 us (6.03 TB/s of
// 6.53), GeGLU of 6,208 x 16,384 93 us (5.5 TB/s), codes of 6,208 x 2,048 8.4 us, of
// one row 1.4 us.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace w4a4 {

enum RowOp : int { kRowQuant = 0, kRowGeglu = 1, kRowNorm = 2 };

// Longest rows held in registers (aligned rows of 8-element vectors).
constexpr int kRow8MaxVec = 32768;

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

// gelu(x) = x / (1 + exp(-2 u)), u = sqrt(2/pi) (x + 0.044715 x^3): the tanh
// form 0.5 x (1 + tanh u) with 1 + tanh u = 2 / (1 + exp(-2 u)), which does not
// cancel for negative u.  exp(-2 u) = 2^(x (a + b x^2)).
constexpr float kGeluA = -2.302208198f;  // -2 sqrt(2/pi) log2(e)
constexpr float kGeluB = -0.1029432397f; // 0.044715 of it
__device__ __forceinline__ float fast_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 gelu_tanh_f32x2(float2 x) {
  const float2 q = __ffma2_rn(make_float2(kGeluB, kGeluB), __fmul2_rn(x, x), make_float2(kGeluA, kGeluA));
  const float2 a = __fmul2_rn(x, q);
  const float2 d = __fadd2_rn(make_float2(fast_ex2(a.x), fast_ex2(a.y)), make_float2(1.f, 1.f));
  return __fmul2_rn(x, make_float2(fast_rcp(d.x), fast_rcp(d.y)));
}

// How codes of a value are formed from a row's scale.  fast: the quotient from
// the reciprocal y, q0 = v y, corrected by its residual, q = q0 + (v - q0 scale) y
// (Markstein, IBM J. Res. Dev. 34, 1990), and rounded by the addition of 1.5 x
// 2^23, whose sum holds the code in its low byte (|v| <= 127.0001 scale, so
// nothing needs a clamp).  Checked for every mantissa of the scale and every v
// within 6 ulp of a tie: q is the quotient that a division rounds to.  q0 alone
// is on the wrong side of ties, of which 16-bit values have many (an element
// that is half of the row's largest).  Measured: 6,208 x 2,048 8.4 us, with q0
// alone 7.7, with a division where one of a thread's values is near a tie 16.0.  Scales
// that are zero, not finite, or whose reciprocal or residual leaves the normal
// numbers are divided by.
struct Coder {
  float mul, div;
  bool fast;
  __device__ __forceinline__ explicit Coder(float scale) {
    const bool finite = scale <= 3.4028234e38f;  // false for NaN
    fast = scale >= 7.8886091e-31f && scale <= 4.2535296e37f;  // 2^-100, 2^125
    mul = fast ? __frcp_rn(scale) : 0.f;
    div = finite && scale > 0.f ? scale : 0.f;
  }
  __device__ __forceinline__ uint32_t slow(float v) const {
    const float t = div > 0.f ? __fdiv_rn(v, div) : 0.f;
    return t == t ? static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(t, -127.f), 127.f))) : 0u;
  }
  // the codes of N values in the low bytes of c
  template <int N>
  __device__ __forceinline__ void codes(const float (&v)[N], uint32_t (&c)[N]) const {
    if (!fast) {
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] = slow(v[i]);
      return;
    }
    constexpr float kMagic = 12582912.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 y = make_float2(mul, mul), x = make_float2(v[i], i + 1 < N ? v[i + 1] : 0.f);
      const float2 q0 = __fmul2_rn(x, y);
      const float2 q = __ffma2_rn(__ffma2_rn(q0, make_float2(-div, -div), x), y, q0);
      const float2 u = __fadd2_rn(q, make_float2(kMagic, kMagic));
      c[i] = __float_as_uint(u.x);
      if (i + 1 < N) c[i + 1] = __float_as_uint(u.y);
    }
  }
};

// Low bytes of four words.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Eight codes.
__device__ __forceinline__ void store_codes(int8_t* p, const float (&v)[8], const Coder& code) {
  uint32_t c[8];
  code.codes(v, c);
  *reinterpret_cast<uint2*>(p) = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
}

// |v| as an unsigned key: ordered like the value, infinity above every finite
// value and NaN above infinity, so a maximum of keys keeps a NaN.
__device__ __forceinline__ uint32_t abs_key(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// max(m, |v|), a NaN of either side kept.
__device__ __forceinline__ float max_abs(float m, float v) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v)));
  return m;
}

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

// Eight elements as they lie in memory, to be asked for early and unpacked later.
template <typename T>
struct RawVec {
  static constexpr int kWords = sizeof(T) / 2;
  uint4 q[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) q[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void unpack(float (&v)[8]) const { load8(reinterpret_cast<const T*>(q), v); }
};

__device__ __forceinline__ void mul8(float (&v)[8], const float (&u)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 r = __fmul2_rn(make_float2(v[i], v[i + 1]), make_float2(u[i], u[i + 1]));
    v[i] = r.x, v[i + 1] = r.y;
  }
}
// v = a v + b
__device__ __forceinline__ void fma8(float (&v)[8], const float (&a)[8], const float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 r = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(v[i], v[i + 1]), make_float2(b[i], b[i + 1]));
    v[i] = r.x, v[i + 1] = r.y;
  }
}
__device__ __forceinline__ void gelu8(float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 r = gelu_tanh_f32x2(make_float2(v[i], v[i + 1]));
    v[i] = r.x, v[i + 1] = r.y;
  }
}

// x and delta / up of 8 elements -> the value before the norm (v + gate u).
template <int OP>
__device__ __forceinline__ void row8_combine(float (&v)[8], float (&u)[8], bool has, bool gated, const float (&gate)[8]) {
  if constexpr (OP == kRowGeglu) {
    gelu8(v);
    mul8(v, u);
  } else if constexpr (OP == kRowNorm) {
    if (has) {
      if (gated) {
        fma8(u, gate, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = u[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += u[i];
      }
    }
  }
}

// One row of a CTA at a time, held in registers: thread t has the 8-element
// groups t, t + blockDim, ... (VPT of them).  A CTA takes consecutive rows, so
// that an observation's gain, shift and gate come from L1 after its first row.
template <typename T, int OP, int VPT, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB) row8_kernel(const __grid_constant__ Row8Params p) {
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[2][32];
  pdl_launch_dependents();
  pdl_wait();
  const int groups = p.h / 8;
  const bool has2 = p.x2 != nullptr;
  RawVec<T> rx[VPT], ru[VPT];
  const auto fetch = [&](long long row) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* x2 = static_cast<const T*>(p.x2) + row * p.ld2;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int g = threadIdx.x + j * blockDim.x;
      if (g < groups) {
        rx[j].load(x + g * 8);
        if (OP != kRowQuant && has2) ru[j].load(x2 + g * 8);
      }
    }
  };
  long long row = p.rows * blockIdx.x / gridDim.x;
  const long long end = p.rows * (blockIdx.x + 1) / gridDim.x;
  fetch(row);
  for (int turn = 0; row < end; ++row, turn ^= 1) {
    const long long obs = OP == kRowNorm ? row / p.rows_per_batch : 0;
    const T* gate = static_cast<const T*>(p.gate) + obs * p.gate_stride;
    float v[VPT][8];
    float ss[2] = {0.f, 0.f};
    {
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int g = threadIdx.x + j * blockDim.x;
        if (g < groups) {
          float u[8];
          rx[j].unpack(v[j]);
          if (OP != kRowQuant && has2) ru[j].unpack(u);
          float gv[8];
          if (OP == kRowNorm && p.gate) load8(gate + g * 8, gv);
          row8_combine<OP>(v[j], u, has2, p.gate != nullptr, gv);
          if constexpr (OP == kRowNorm) {
            if (p.total) store8(static_cast<T*>(p.total) + row * p.h + g * 8, v[j]);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss[i & 1] = fmaf(v[j][i], v[j][i], ss[i & 1]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
        }
      }
    }
    if (row + 1 < end) fetch(row + 1);
    if constexpr (OP == kRowNorm) {
      const float rstd = rsqrtf(block_sum(ss[0] + ss[1], red_sum) / static_cast<float>(p.h) + p.eps);
      const float* gain = p.gain + obs * p.gain_stride;
      const float* shift = p.shift + obs * p.shift_stride;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int g = threadIdx.x + j * blockDim.x;
        if (g < groups) {
          float gn[8], sh[8], r[8];
          load8(gain + g * 8, gn);
#pragma unroll
          for (int i = 0; i < 8; ++i) r[i] = rstd, sh[i] = 0.f;
          if (p.shift) load8(shift + g * 8, sh);
          mul8(v[j], r);
          fma8(v[j], gn, sh);
        }
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = max_abs(amax, v[j][i]);
    const float scale = __uint_as_float(block_max(abs_key(amax), red_max[turn])) * kInv127;
    const Coder code(scale);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int g = threadIdx.x + j * blockDim.x;
      if (g < groups) store_codes(p.codes + row * p.ldc + g * 8, v[j], code);
    }
    if (threadIdx.x == 0) p.scale[row] = scale;
  }
}

// Any row: one, two or four elements at a time, the row's fp32 values in shared
// memory between the passes.  For rows that do not begin at multiples of 16
// bytes (a length that is not a multiple of 8), and for long ones.  Bound by the
// instructions and latency of the narrow loads: 1,944 x 7,620 (by 4) 40 us, 4,464 x
// 2,394 (by 2) 33 us, 6,208 x 2,047 codes (by 1) 29 us.  Vectors of 16 bytes from
// the last multiple of 16 before each row on took 17 us for these codes, but 40
// and 63 us for the two norms, whose operands lie differently; several steps'
// loads at once took 42 us for 4,464 x 2,394.
constexpr int kRow8AnyThreads = 256;
constexpr int kRow8AnyMax = 49152;  // elements: 192 KB of shared memory

// W = 4, 2 or 1 elements, aligned to their size.
template <int W, typename T>
__device__ __forceinline__ void load_few(const T* p, float (&v)[W]) {
  struct alignas(W * sizeof(T)) Pack { T x[W]; };
  const Pack a = *reinterpret_cast<const Pack*>(p);
#pragma unroll
  for (int i = 0; i < W; ++i) v[i] = to_float(a.x[i]);
}
template <int W, typename T>
__device__ __forceinline__ void store_few(T* p, const float (&v)[W]) {
  struct alignas(W * sizeof(T)) Pack { T x[W]; };
  Pack a;
#pragma unroll
  for (int i = 0; i < W; ++i) a.x[i] = from_float<T>(v[i]);
  *reinterpret_cast<Pack*>(p) = a;
}

template <typename T, int OP, int W>
__global__ void __launch_bounds__(kRow8AnyThreads) row8_any_kernel(const __grid_constant__ Row8Params p) {
  extern __shared__ __align__(16) float row8_smem[];
  __shared__ float red_sum[32];
  __shared__ uint32_t red_max[32];
  pdl_launch_dependents();
  pdl_wait();
  const long long row = blockIdx.x;
  const long long obs = OP == kRowNorm ? row / p.rows_per_batch : 0;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* x2 = p.x2 ? static_cast<const T*>(p.x2) + row * p.ld2 : nullptr;
  const T* gate = p.gate ? static_cast<const T*>(p.gate) + obs * p.gate_stride : nullptr;
  float ss = 0.f, amax = 0.f;
#pragma unroll 4
  for (int e = W * threadIdx.x; e < p.h; e += W * blockDim.x) {
    float v[W], u[W], g[W];
    load_few<W>(x + e, v);
    if (OP != kRowQuant && x2) load_few<W>(x2 + e, u);
    if (OP == kRowNorm && gate) load_few<W>(gate + e, g);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (OP == kRowGeglu) v[i] = gelu_tanh_f32x2(make_float2(v[i], 0.f)).x * u[i];
      if constexpr (OP == kRowNorm) {
        if (x2) v[i] = gate ? fmaf(g[i], u[i], v[i]) : v[i] + u[i];
        ss = fmaf(v[i], v[i], ss);
      } else {
        amax = max_abs(amax, v[i]);
      }
    }
    if (OP == kRowNorm && p.total) store_few<W>(static_cast<T*>(p.total) + row * p.h + e, v);
    store_few<W>(row8_smem + e, v);
  }
  if constexpr (OP == kRowNorm) {
    const float rstd = rsqrtf(block_sum(ss, red_sum) / static_cast<float>(p.h) + p.eps);
    const float* gain = p.gain + obs * p.gain_stride;
    const float* shift = p.shift ? p.shift + obs * p.shift_stride : nullptr;
#pragma unroll 4
    for (int e = W * threadIdx.x; e < p.h; e += W * blockDim.x) {
      float v[W], g[W], b[W];
      load_few<W>(row8_smem + e, v);
      load_few<W>(gain + e, g);
#pragma unroll
      for (int i = 0; i < W; ++i) b[i] = 0.f;
      if (shift) load_few<W>(shift + e, b);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        v[i] = fmaf(v[i] * rstd, g[i], b[i]);
        amax = max_abs(amax, v[i]);
      }
      store_few<W>(row8_smem + e, v);
    }
  }
  const float scale = __uint_as_float(block_max(abs_key(amax), red_max)) * kInv127;
  const Coder code(scale);
#pragma unroll 4
  for (int e = W * threadIdx.x; e < p.h; e += W * blockDim.x) {
    struct alignas(W) Bytes { int8_t x[W]; } bytes;
    float v[W];
    uint32_t c[W];
    load_few<W>(row8_smem + e, v);
    code.codes(v, c);
#pragma unroll
    for (int i = 0; i < W; ++i) bytes.x[i] = static_cast<int8_t>(c[i]);
    *reinterpret_cast<Bytes*>(p.codes + row * p.ldc + e) = bytes;
  }
  if (threadIdx.x == 0) p.scale[row] = scale;
}

// Elements from the last multiple of 16 bytes before p to p.
template <typename T>
__device__ __forceinline__ int row_lead(const T* p) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

// out[r, :] = codes[r, :] * scale[r], rounded once; grid (column groups, rows).
// VEC: 16 codes a thread, of rows of codes and results that begin at multiples
// of 16 bytes.  Otherwise a thread writes one 16-byte vector of the results,
// whose codes it cuts out of the words around them (rows of codes at multiples
// of 4 bytes; else, and at the row's ends, by elements): 4,464 x 2,394 in 11 us,
// by elements in 47.  Bound: HBM; 6,208 x 2,048 7.9 us (4.8 TB/s).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dequant8_kernel(const int8_t* __restrict__ codes, long long ldc,
                                                       const float* __restrict__ scale, T* __restrict__ out,
                                                       long long rows, int h) {
  pdl_launch_dependents();
  pdl_wait();
  const int at = blockIdx.x * blockDim.x + threadIdx.x;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    const int8_t* src = codes + row * ldc;
    T* dst = out + row * h;
    if constexpr (VEC) {
      const int e = 16 * at;
      if (e >= h) return;
      const float s = __ldg(scale + row);
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src + e));
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = static_cast<float>(static_cast<int8_t>(w[2 * half + (j >> 2)] >> (8 * (j & 3)))) * s;
        store8(dst + e + 8 * half, v);
      }
    } else {
      constexpr int E = 16 / sizeof(T);
      const int e = E * at - row_lead(dst);
      if (e >= h) continue;
      const float s = __ldg(scale + row);
      float v[E];
      if (e >= 0 && e + E <= h && (reinterpret_cast<uintptr_t>(src) & 3) == 0) {
        const uint32_t* words = reinterpret_cast<const uint32_t*>(src + (e & ~3));
        const int cut = e & 3;
        uint32_t w[E / 4 + 1];
#pragma unroll
        for (int i = 0; i < E / 4; ++i) w[i] = __ldg(words + i);
        w[E / 4] = cut ? __ldg(words + E / 4) : 0u;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const uint32_t four = __funnelshift_r(w[j / 4], w[j / 4 + 1], 8 * cut);
          v[j] = static_cast<float>(static_cast<int8_t>(four >> (8 * (j & 3)))) * s;
        }
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = e + j >= 0 && e + j < h ? static_cast<float>(src[e + j]) * s : 0.f;
      }
      if (e >= 0 && e + E <= h) {
        uint4 whole;
        T* y = reinterpret_cast<T*>(&whole);
#pragma unroll
        for (int j = 0; j < E; ++j) y[j] = from_float<T>(v[j]);
        *reinterpret_cast<uint4*>(dst + e) = whole;
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (e + j >= 0 && e + j < h) dst[e + j] = from_float<T>(v[j]);
      }
    }
  }
}

}  // namespace w4a4
