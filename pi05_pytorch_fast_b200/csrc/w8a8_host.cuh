// Launchers and C entry points of the 8-bit serving operators (rows8.cuh,
// gemm8.cuh, kv8.cuh, attention8.cuh).  Included by w4a4_sm100.cu, whose
// helpers (fail, launch_kernel, make_map, ...) it uses.
#pragma once

#include "attention8.cuh"
#include "gemm8.cuh"
#include "kv8.cuh"
#include "rows8.cuh"

namespace w4a4 {
namespace {

// No kernel with TMEM fits beside one of these on an SM (kOneCtaSmem).
constexpr int kSmSharedMemory = 228 * 1024, kCtaReserved = 1024;
constexpr bool fits_beside(int bytes) { return kOneCtaSmem + bytes + 2 * kCtaReserved <= kSmSharedMemory; }
static_assert(!fits_beside(kOneCtaSmem) && !fits_beside(gemm_smem_bytes(16)) && !fits_beside(gemm_pair_smem_bytes(16)) &&
                  !fits_beside(gemm_pair_i8_smem_bytes(16)) && !fits_beside(kAttnSmem),
              "a kernel with TMEM could share an SM with an 8-bit one");
static_assert(gemm8_tile_smem(16, 1, false) >= kOneCtaSmem && kG8PairSmem >= kOneCtaSmem &&
                  Attn8Many<64>::kSmem >= kOneCtaSmem && Attn8Many<256>::kSmem >= kOneCtaSmem,
              "every 8-bit kernel with TMEM has its SM to itself");

// Calls f with a value of the element type that `dtype` names.
template <class F>
int by_dtype(int32_t dtype, bool fp32_too, const char* what, F f) {
  switch (dtype) {
    case W4A4_F16: return f(__half{});
    case W4A4_BF16: return f(__nv_bfloat16{});
    case W4A4_F32:
      if (fp32_too) return f(float{});
      break;
    default: break;
  }
  return fail(W4A4_ERR_INVALID, "%s: unsupported dtype code %d", what, dtype);
}

int elem_size(int32_t dtype) { return dtype == W4A4_F32 ? 4 : 2; }

// Kernels of this file whose dynamic shared memory has been raised, by device
// and number.
uint64_t g_attr8_done[kMaxDevices];
template <class Kernel>
int ensure_smem_attr8(int dev, int bit, Kernel kernel, int bytes) {
  std::lock_guard<std::mutex> lk(g_dev_mu);
  if (!(g_attr8_done[dev] >> bit & 1)) {
    W4A4_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    g_attr8_done[dev] |= 1ull << bit;
  }
  return W4A4_OK;
}

// Tiled map of rank 2 to 4, zeros outside, encoded for each call: dims[0]
// innermost (elements), strides_bytes[i] the byte stride of dims[i + 1].
int encode_map(CUtensorMap* out, const void* ptr, CUtensorMapDataType type, int rank, const uint64_t* dims,
               const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(W4A4_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
  cuuint64_t d[4], st[3];
  cuuint32_t bx[4], one[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i], bx[i] = box[i];
    if (i + 1 < rank) st[i] = strides_bytes[i];
  }
  const CUresult r = fn(out, type, static_cast<cuuint32_t>(rank), const_cast<void*>(ptr), d, st, bx, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? W4A4_OK
                           : fail(W4A4_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d): rank %d, inner %llu, rows %llu, stride %llu",
                                  static_cast<int>(r), rank, (unsigned long long)d[0], (unsigned long long)d[1],
                                  (unsigned long long)st[0]);
}

// Whether rows of `stride` elements of `size` bytes from p all begin at a
// multiple of `bytes`.
bool rows_aligned(const void* p, int64_t stride, int size, int bytes) {
  return aligned(p, bytes) && (stride * size) % bytes == 0;
}

template <int OP>
int launch_row8(Row8Params p, int32_t dtype, cudaStream_t stream, const char* what) {
  if (p.rows == 0) return ok();
  if (p.rows > 0x7fffffffLL) return fail(W4A4_ERR_UNSUPPORTED, "%s: too many rows: %lld", what, (long long)p.rows);
  const int size = elem_size(dtype);
  // The 8-element path wants 16-byte vectors of every operand and 8-byte
  // vectors of codes.
  bool vec = p.h % 8 == 0 && rows_aligned(p.x, p.ldx, size, 16) && rows_aligned(p.codes, p.ldc, 1, 8);
  if (p.x2) vec = vec && rows_aligned(p.x2, p.ld2, size, 16);
  if (p.gate) vec = vec && rows_aligned(p.gate, p.gate_stride, size, 16);
  if (p.gain) vec = vec && rows_aligned(p.gain, p.gain_stride, 4, 16);
  if (p.shift) vec = vec && rows_aligned(p.shift, p.shift_stride, 4, 16);
  if (p.total) vec = vec && aligned(p.total, 16);
  return by_dtype(dtype, true, what, [&](auto tag) {
    using T = decltype(tag);
    int dev, sms;
    if (int e = current_device(&dev)) return e;
    if (int e = sm_count(dev, &sms)) return e;
    // as many CTAs as run at once (2,048 threads and 64 K registers of an SM), each with its share of the rows
    const auto go = [&](void (*kernel)(const Row8Params), int groups, int vpt, int regs) {
      const int threads = (((groups + vpt - 1) / vpt) + 31) / 32 * 32;
      const int ctas = std::max(1, std::min({2048 / threads, 65536 / (threads * regs), 32}));
      const dim3 grid(static_cast<unsigned>(std::min<int64_t>(p.rows, static_cast<int64_t>(sms) * ctas)));
      return cuda_status(launch_kernel(kernel, grid, dim3(threads), 0, stream, 1, p)) ? W4A4_ERR_CUDA : ok();
    };
    if (vec && p.h <= kRow8MaxVec) {
      const int groups = p.h / 8;
      // few rows: as many threads as a row has vectors, for the latency (400 x 1,024: 2.9 us, with four vectors a thread
      // 3.4); many: four vectors a thread, so that the reductions' instructions are shared by more elements (776 x 2,048:
      // 4.5 us against 5.1; 49,664 x 2,048: 115 against 140)
      if (groups <= 256 && p.rows <= 4 * sms) return go(row8_kernel<T, OP, 1, 256, 4>, groups, 1, 64);
      if (groups <= 64) return go(row8_kernel<T, OP, 2, 512, 1>, groups, 2, 128);
      if (groups <= 2048) return go(row8_kernel<T, OP, 4, 512, 1>, groups, 4, 128);
      return go(row8_kernel<T, OP, 4, 1024, 1>, groups, 4, 64);
    }
    if (p.h > kRow8AnyMax)
      return fail(W4A4_ERR_UNSUPPORTED, "%s: rows of more than %d elements are not supported", what, kRow8AnyMax);
    // elements at a time: what the length and every operand's rows allow
    const auto together = [&](int w) {
      bool fits = p.h % w == 0 && rows_aligned(p.x, p.ldx, size, w * size) && rows_aligned(p.codes, p.ldc, 1, w);
      if (p.x2) fits = fits && rows_aligned(p.x2, p.ld2, size, w * size);
      if (p.gate) fits = fits && rows_aligned(p.gate, p.gate_stride, size, w * size);
      if (p.gain) fits = fits && rows_aligned(p.gain, p.gain_stride, 4, w * 4);
      if (p.shift) fits = fits && rows_aligned(p.shift, p.shift_stride, 4, w * 4);
      if (p.total) fits = fits && aligned(p.total, w * size);
      return fits;
    };
    const int w = together(4) ? 2 : together(2) ? 1 : 0;
    const auto kernel = w == 2 ? row8_any_kernel<T, OP, 4> : w == 1 ? row8_any_kernel<T, OP, 2> : row8_any_kernel<T, OP, 1>;
    const int bytes = p.h * 4;
    if (bytes > 40 * 1024) {
      const int bit = 32 + w + 3 * OP + 9 * (std::is_same_v<T, float> ? 0 : std::is_same_v<T, __half> ? 1 : 2);
      if (int e = ensure_smem_attr8(dev, bit, kernel, kRow8AnyMax * 4)) return e;
    }
    // four steps of a row a thread, up to 256 threads
    const int each = 4 << w, threads = std::min(kRow8AnyThreads, ((p.h + each - 1) / each + 31) / 32 * 32);
    return cuda_status(launch_kernel(kernel, dim3(static_cast<unsigned>(p.rows)), dim3(threads), bytes, stream, 1, p))
               ? W4A4_ERR_CUDA
               : ok();
  });
}

int check_rows8(int64_t rows, int32_t h, const void* x, int64_t ldx, const int8_t* codes, int64_t ldc,
                const float* scale, const char* what) {
  if (rows < 0 || h <= 0) return fail(W4A4_ERR_INVALID, "%s: invalid shape [%lld, %d]", what, (long long)rows, h);
  if (rows == 0) return W4A4_OK;
  if (!x || !codes || !scale) return fail(W4A4_ERR_INVALID, "%s: null pointer argument", what);
  if (ldx < h || ldc < h) return fail(W4A4_ERR_INVALID, "%s: row stride below %d", what, h);
  return W4A4_OK;
}

// How a product of more than 16 tokens runs: on CTA pairs, or in tiles of 128
// channels x tok_tile tokens whose K is split over clusters of `split` CTAs.
struct Gemm8Plan {
  bool pair;
  int tok_tile, split, stages;
  int n_tok_tiles, n_w_tiles;
};

// The cheapest of the two kernels' launch shapes, by a model in us fitted to
// graph-timed runs on a B200 of 30 shapes (17 .. 2,048 tokens, K 64 .. 16,384, N 64
// .. 16,384) in every shape that the kernels allow:
//   tile: a wave costs 4.0 + 0.012 T (set-up, first loads, epilogue) and a step
//   of K 0.16 + 0.0006 T; splitting K adds 1.2 + 0.012 T for the exchange;
//   pair: 6.0, and a wave its steps at 0.27 or its epilogue at 2.4.
// The choice is within 8 % of the best measured shape for 27 of them.  One
// CTA runs on an SM; `fit[i]` is how many clusters of 1 << i CTAs fit the
// device at once (148, 74, 33 and 15 on a B200: whole clusters in a GPC).
Gemm8Plan gemm8_plan(int64_t m, int n, int k, const int (&fit)[4]) {
  Gemm8Plan best{};
  double cost = 1e300;
  const int k_steps = (k + 127) / 128;
  const auto waves = [](int64_t tiles, int at_once) { return static_cast<double>((tiles + at_once - 1) / at_once); };
  const int n_w_tiles = (n + 127) / 128;
  // fewer token tiles than this would exceed 256 tokens, more would be below 16
  const int64_t most = std::min<int64_t>((m + 15) / 16, (m + 255) / 256 + 64);
  for (int64_t tiles = (m + 255) / 256; tiles <= most; ++tiles) {
    const int t = static_cast<int>(((m + tiles - 1) / tiles + 15) / 16 * 16);
    const int n_tok_tiles = static_cast<int>((m + t - 1) / t);
    for (int i = 0; i < 4; ++i) {
      const int split = 1 << i;
      if (fit[i] < 1 || (split > 1 && (split > k_steps || t > 128))) continue;
      const int steps = (k_steps + split - 1) / split;
      const double c = waves(static_cast<int64_t>(n_tok_tiles) * n_w_tiles, fit[i]) * (4.0 + 0.012 * t + steps * (0.16 + 0.0006 * t)) +
                       (split > 1 ? 1.2 + 0.012 * t : 0.0);
      if (c < cost - 1e-9) {
        cost = c;
        best = {false, t, split, 0, n_tok_tiles, n_w_tiles};
      }
    }
  }
  const int64_t pair_tiles = ((m + 255) / 256) * ((n + 255) / 256);
  if (6.0 + waves(pair_tiles, fit[1]) * std::max(0.27 * k_steps, 2.4) < cost) {
    best = {true, 0, 1, 0, static_cast<int>((m + 255) / 256), (n + 255) / 256};
    return best;
  }
  const int steps = (k_steps + best.split - 1) / best.split;
  best.stages = std::max(1, std::min({steps, kG8MaxStages, 200 * 1024 / (kG8ABytes + best.tok_tile * kG8StepBytes)}));
  return best;
}

// The launch shape for up to 16 tokens.  16 channels a CTA where that leaves enough CTAs (the tokens are read half as
// often; 1 x 2,048 x 32,768: 17.1 us, with 8 channels 19.0), and twice the warps, to have enough loads under way, where
// there are few CTAs and a long K (16 x 16,384 x 2,048: 9.6 us, with 8 warps 16.1); half the MMA's rows for up to 8 tokens
// (1 x 16,384 x 2,048: 11.6 us, with all of them and 8 warps 14.8).
struct Gemm8FewPlan {
  bool half, wide, deep;
  int ctas, threads;
};
Gemm8FewPlan gemm8_few_plan(int64_t m, int n, int k, int sms) {
  const bool wide = n >= 32 * sms, deep = !wide && k >= 4096;
  const int per = wide ? 16 : 8;
  return {m <= 8, wide, deep, (n + per - 1) / per, deep ? 512 : 256};
}

// Clusters of 1, 2, 4 and 8 CTAs that the device runs at once with one CTA to an SM.
int g_cluster_fit[kMaxDevices][4];
int cluster_fit(int dev, int (&fit)[4]) {
  int sms;
  if (int e = sm_count(dev, &sms)) return e;
  std::lock_guard<std::mutex> lk(g_dev_mu);
  int(&f)[4] = g_cluster_fit[dev];
  if (f[0] == 0) {
    W4A4_CUDA_TRY(cudaFuncSetAttribute(gemm8_tile_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit));
    for (int i = 1; i < 4; ++i) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1u << i;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(8 << i);
      cfg.blockDim = dim3(kG8TileThreads);
      cfg.dynamicSmemBytes = kOneCtaSmem;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      W4A4_CUDA_TRY(cudaOccupancyMaxActiveClusters(&f[i], gemm8_tile_kernel<__half>, &cfg));
    }
    f[0] = sms;
  }
  std::copy(f, f + 4, fit);
  return W4A4_OK;
}

int gemm8_codes_map(CUtensorMap* out, const int8_t* ptr, int k, int64_t rows, int64_t ld, int box) {
  const uint64_t dims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows)}, stride = static_cast<uint64_t>(ld);
  const uint32_t boxes[2] = {128, static_cast<uint32_t>(box)};
  return encode_map(out, ptr, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, dims, &stride, boxes, CU_TENSOR_MAP_SWIZZLE_128B);
}

int launch_gemm8(const int8_t* a, int64_t lda, const float* sa, const int8_t* w, int64_t ldw, const float* sw,
                 const void* bias, int32_t dtype, int64_t m, int32_t n, int32_t k, void* y, cudaStream_t stream) {
  int dev, sms;
  if (int e = current_device(&dev)) return e;
  if (int e = sm_count(dev, &sms)) return e;
  if (m <= kG8FewTokens) {
    const Gemm8FewParams f{a, w, sa, sw, bias, y, lda, ldw, static_cast<int>(m), n, k};
    return by_dtype(dtype, true, "gemm8", [&](auto tag) {
      using T = decltype(tag);
      const Gemm8FewPlan plan = gemm8_few_plan(m, n, k, sms);
      const auto by_shape = [&](auto half_tag) {
        constexpr bool H = decltype(half_tag)::value;
        return plan.deep   ? gemm8_few_kernel<T, H, 1, 16>
               : plan.wide ? gemm8_few_kernel<T, H, 2, 8>
                           : gemm8_few_kernel<T, H, 1, 8>;
      };
      const auto kernel = plan.half ? by_shape(std::true_type{}) : by_shape(std::false_type{});
      W4A4_CUDA_TRY(launch_kernel(kernel, dim3(plan.ctas), dim3(plan.threads), 0, stream, 1, f));
      return ok();
    });
  }
  int fit[4];
  if (int e = cluster_fit(dev, fit)) return e;
  const Gemm8Plan plan = gemm8_plan(m, n, k, fit);
  Gemm8Params p;
  if (int e = gemm8_codes_map(&p.tmap_a, a, k, m, lda, plan.pair ? 128 : plan.tok_tile)) return e;
  if (int e = gemm8_codes_map(&p.tmap_w, w, k, n, ldw, 128)) return e;
  p.sa = sa, p.sw = sw, p.bias = bias, p.y = y, p.m = m, p.n = n;
  p.k_steps = (k + 127) / 128, p.tok_tile = plan.tok_tile, p.stages = plan.stages;
  p.n_tok_tiles = plan.n_tok_tiles, p.n_w_tiles = plan.n_w_tiles, p.wait_limit_ns = g_wait_limit_ns.load();
  return by_dtype(dtype, true, "gemm8", [&](auto tag) {
    using T = decltype(tag);
    const int bit = 24 + 2 * (std::is_same_v<T, float> ? 0 : std::is_same_v<T, __half> ? 1 : 2);
    if (plan.pair) {
      p.tma_store = n * sizeof(T) % 16 == 0;
      if (p.tma_store) {
        const auto type = std::is_same_v<T, float>    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                          : std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        const uint64_t dims[2] = {static_cast<uint64_t>(n), static_cast<uint64_t>(m)}, stride = n * sizeof(T);
        const uint32_t box[2] = {64 / sizeof(T), 32};
        if (int e = encode_map(&p.tmap_y, y, type, 2, dims, &stride, box, CU_TENSOR_MAP_SWIZZLE_64B)) return e;
      }
      if (int e = ensure_smem_attr8(dev, bit, gemm8_pair_kernel<T>, kG8PairSmem)) return e;
      const int pairs = std::min(sms / 2, plan.n_tok_tiles * plan.n_w_tiles);
      W4A4_CUDA_TRY(launch_kernel(gemm8_pair_kernel<T>, dim3(2 * pairs), dim3(kG8PairThreads), kG8PairSmem, stream, 2, p));
    } else {
      if (int e = ensure_smem_attr8(dev, bit + 1, gemm8_tile_kernel<T>, kSmemLimit)) return e;
      W4A4_CUDA_TRY(launch_kernel(gemm8_tile_kernel<T>, dim3(plan.split * plan.n_tok_tiles * plan.n_w_tiles),
                                  dim3(kG8TileThreads), gemm8_tile_smem(plan.tok_tile, plan.stages, plan.split > 1), stream, plan.split, p));
    }
    return ok();
  });
}

// Shape and layout of a cache: width 64, 128 or 256, capacity a
// multiple of 16, strides and bases multiples of 16 bytes.
int check_cache8(const void* k, const void* v, const void* ks, const void* vs, const int64_t* stride, int32_t batch,
                 int32_t heads, int32_t width, int32_t capacity, const char* what) {
  if (batch < 0 || heads <= 0) return fail(W4A4_ERR_INVALID, "%s: invalid batch %d or heads %d", what, batch, heads);
  if (width != 64 && width != 128 && width != 256)
    return fail(W4A4_ERR_UNSUPPORTED, "%s: head width must be 64, 128 or 256, got %d", what, width);
  if (capacity <= 0 || capacity % kKvBlock)
    return fail(W4A4_ERR_INVALID, "%s: the capacity must be a positive multiple of %d, got %d", what, kKvBlock, capacity);
  if (static_cast<int64_t>(batch) * heads > 65535)
    return fail(W4A4_ERR_UNSUPPORTED, "%s: batch x heads must be at most 65535, got %d x %d", what, batch, heads);
  if (!stride) return fail(W4A4_ERR_INVALID, "%s: null pointer argument", what);
  if (batch == 0) return W4A4_OK;
  if (!k || !v || !ks || !vs) return fail(W4A4_ERR_INVALID, "%s: null pointer argument", what);
  if (!aligned(k, 16) || !aligned(v, 16) || stride[0] % 16 || stride[1] % 16 || stride[2] % 16)
    return fail(W4A4_ERR_INVALID, "%s: cache rows must begin at multiples of 16 bytes", what);
  if (stride[0] < width || stride[1] < width || stride[2] < width)
    return fail(W4A4_ERR_INVALID, "%s: cache strides must be at least the head width", what);
  return W4A4_OK;
}

// How many CTAs the keys of one key/value head are split over, from the
// cache's capacity (the lengths are on the device; a split without keys writes
// an empty part).  Up to 8 CTAs of the few-rows form are a cluster, as long as
// all clusters run at once: `fit[i]` of 1 << i CTAs; they join their parts
// themselves (8 heads of width 256 over 776 tokens: 7.5 us, 10.2 with the parts
// in memory and a kernel that joins them).
//
// The few-rows form is for up to 16 rows, its MMA's; the other one pads them to
// 128 (8 rows, 776 tokens of width 256: 7.5 and 14.8 us; 16 rows, 65,536 tokens
// of 4 x 2 heads of width 128: 41 and 102 us).
constexpr int kAttn8FewRows = 16;
struct Attn8Plan {
  bool few;
  int tiles;   // row tiles of the many-rows form
  int splits;
};
Attn8Plan attn8_plan(int64_t units, int64_t rows, int capacity, int width, const int (&fit)[4]) {
  Attn8Plan plan{};
  plan.few = rows <= kAttn8FewRows;
  plan.tiles = static_cast<int>((rows + 127) / 128);
  const int64_t work = units * (plan.few ? 1 : plan.tiles);
  // splits that the keys are worth (one step of all 8 warps, or three tiles of 64 keys, each) and that the SMs have
  // room for, at most 128 of them and the steps in equal shares, as each part costs the join (1 head of 256, 32,768
  // tokens: 128 parts 14.7 us, 148 parts 20.9, 64 parts 15.7; 131,072 tokens: 26.5, 31.8 and 35.4)
  const int step = plan.few ? 32768 / width : 192;
  const int64_t steps = (capacity + step - 1) / step;
  const int64_t room = std::max<int64_t>(1, std::min<int64_t>(128, fit[0] / std::max<int64_t>(work, 1)));
  const int64_t each = (steps + room - 1) / room;
  plan.splits = static_cast<int>(plan.few ? (steps + each - 1) / each : std::min(steps, room));
  if (plan.few && plan.splits <= 8) {
    // a cluster of 3, 5, 6 or 7 takes no more room than one of the next power of two
    const auto room_for = [&](int splits) { return fit[splits > 4 ? 3 : splits > 2 ? 2 : splits - 1]; };
    while (plan.splits > 1 && units > room_for(plan.splits)) --plan.splits;
  }
  return plan;
}

template <typename T, int D>
int launch_attention8_d(const Attn8Params& p, const Attn8Plan& plan, int64_t units, int dev, int bit,
                        cudaStream_t stream) {
  if (plan.few) {
    const auto go = [&](auto half_tag, int nr) {
      constexpr bool HALF = decltype(half_tag)::value;
      using C = Attn8Few<D, HALF>;
      const auto kernel = attn8_few_kernel<T, D, HALF>;
      if (int e = ensure_smem_attr8(dev, nr, kernel, C::kSmem)) return e;
      // up to 8 CTAs of a key/value head form a cluster and join their parts themselves
      W4A4_CUDA_TRY(launch_kernel(kernel, dim3(p.splits, static_cast<unsigned>(units)), dim3(C::kThreads), C::kSmem,
                                  stream, p.splits <= 8 ? p.splits : 1, p));
      return static_cast<int>(W4A4_OK);
    };
    if (int e = p.rows <= 8 ? go(std::true_type{}, bit) : go(std::false_type{}, bit + 1)) return e;
  } else {
    using C = Attn8Many<D>;
    const auto kernel = attn8_many_kernel<T, D>;
    // the register split draws on what the CTA is launched with: more than that would wait for good
    static const int regs = [&] {
      cudaFuncAttributes fa;
      return cudaFuncGetAttributes(&fa, kernel) == cudaSuccess ? (fa.numRegs + 7) / 8 * 8 : 0;
    }();
    if (regs * C::kThreads < C::kPoolRegs)
      return fail(W4A4_ERR_UNSUPPORTED, "attention8: built with %d registers a thread, too few for its register split", regs);
    if (int e = ensure_smem_attr8(dev, bit + 2, kernel, C::kSmem)) return e;
    Attn8ManyParams mp;
    mp.p = p;
    const uint64_t dims[4] = {D, static_cast<uint64_t>(p.heads), static_cast<uint64_t>(p.capacity),
                              static_cast<uint64_t>(units / p.heads)};
    const uint64_t strides[3] = {static_cast<uint64_t>(p.ch), static_cast<uint64_t>(p.ct), static_cast<uint64_t>(p.cb)};
    const uint32_t box[4] = {D < 128 ? D : 128, 1, C::kKeys, 1};
    const CUtensorMapSwizzle sw = D < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    if (int e = encode_map(&mp.tmap_k, p.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, dims, strides, box, sw)) return e;
    if (int e = encode_map(&mp.tmap_v, p.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, dims, strides, box, sw)) return e;
    W4A4_CUDA_TRY(launch_kernel(kernel, dim3(plan.tiles, p.splits, static_cast<unsigned>(units)), dim3(C::kThreads), C::kSmem,
                                stream, 1, mp));
  }
  if (p.splits > (plan.few ? 8 : 1)) {
    const bool wide = p.splits > 32;
    W4A4_CUDA_TRY(launch_kernel(wide ? attn8_join_kernel<T, D, 512> : attn8_join_kernel<T, D, 128>,
                                dim3(static_cast<unsigned>(p.rows), static_cast<unsigned>(units)), dim3(wide ? 512 : 128), 0,
                                stream, 1, p));
  }
  return ok();
}

int launch_attention8(const Attn8Params& p, const Attn8Plan& plan, int64_t units, int width, int32_t dtype, int dev,
                      cudaStream_t stream) {
  return by_dtype(dtype, false, "attention8", [&](auto tag) {
    using T = decltype(tag);
    if constexpr (std::is_same_v<T, float>) return fail(W4A4_ERR_INVALID, "attention8: unsupported dtype");
    else {
      const int bit = std::is_same_v<T, __half> ? 0 : 12;
      switch (width) {
        case 64: return launch_attention8_d<T, 64>(p, plan, units, dev, bit, stream);
        case 128: return launch_attention8_d<T, 128>(p, plan, units, dev, bit + 4, stream);
        default: return launch_attention8_d<T, 256>(p, plan, units, dev, bit + 8, stream);
      }
    }
  });
}

}  // namespace
}  // namespace w4a4

extern "C" {

int w4a4_rms_norm_quant8(const void* x, int64_t ldx, const void* delta, int64_t ldd, const void* gate,
                         int64_t gate_stride, const float* gain, int64_t gain_stride, const float* shift,
                         int64_t shift_stride, float eps, int32_t dtype, int64_t rows, int32_t rows_per_batch,
                         int32_t h, void* total, int8_t* codes, int64_t ldc, float* scale, void* stream) {
  if (int e = check_rows8(rows, h, x, ldx, codes, ldc, scale, "rms_norm_quant8")) return e;
  if (rows_per_batch <= 0) return fail(W4A4_ERR_INVALID, "rms_norm_quant8: rows_per_batch must be positive");
  if (rows > 0 && !gain) return fail(W4A4_ERR_INVALID, "rms_norm_quant8: null pointer argument");
  if (delta && ldd < h) return fail(W4A4_ERR_INVALID, "rms_norm_quant8: row stride below %d", h);
  if (gate && !delta) return fail(W4A4_ERR_INVALID, "rms_norm_quant8: a gate needs a delta");
  if (gate_stride < 0 || gain_stride < 0 || shift_stride < 0)
    return fail(W4A4_ERR_INVALID, "rms_norm_quant8: negative stride");
  Row8Params p{};
  p.x = x, p.ldx = ldx, p.x2 = delta, p.ld2 = ldd;
  p.gate = gate, p.gate_stride = gate_stride, p.gain = gain, p.gain_stride = gain_stride;
  p.shift = shift, p.shift_stride = shift_stride;
  p.total = total, p.codes = codes, p.ldc = ldc, p.scale = scale;
  p.rows = rows, p.rows_per_batch = rows_per_batch, p.h = h, p.eps = eps;
  return launch_row8<kRowNorm>(p, dtype, static_cast<cudaStream_t>(stream), "rms_norm_quant8");
}

int w4a4_quant8(const void* x, int64_t ldx, const void* up, int64_t ldu, int32_t dtype, int64_t rows, int32_t h,
                int8_t* codes, int64_t ldc, float* scale, void* stream) {
  if (int e = check_rows8(rows, h, x, ldx, codes, ldc, scale, "quant8")) return e;
  if (up && ldu < h) return fail(W4A4_ERR_INVALID, "quant8: row stride below %d", h);
  Row8Params p{};
  p.x = x, p.ldx = ldx, p.x2 = up, p.ld2 = ldu;
  p.codes = codes, p.ldc = ldc, p.scale = scale;
  p.rows = rows, p.rows_per_batch = 1, p.h = h;
  return up ? launch_row8<kRowGeglu>(p, dtype, static_cast<cudaStream_t>(stream), "quant8")
            : launch_row8<kRowQuant>(p, dtype, static_cast<cudaStream_t>(stream), "quant8");
}

int w4a4_dequant8(const int8_t* codes, int64_t ldc, const float* scale, int32_t dtype, int64_t rows, int32_t h,
                  void* out, void* stream) {
  if (int e = check_rows8(rows, h, out, h, codes, ldc, scale, "dequant8")) return e;
  if (rows == 0) return ok();
  const bool vec = h % 16 == 0 && rows_aligned(codes, ldc, 1, 16) && aligned(out, 16);
  return by_dtype(dtype, true, "dequant8", [&](auto tag) {
    using T = decltype(tag);
    const int each = vec ? 16 : 16 / static_cast<int>(sizeof(T));
    const int groups = (h + each - 1) / each + !vec;  // one more where a row may begin inside its first vector
    const int threads = std::min(256, (groups + 31) / 32 * 32);
    const dim3 grid((groups + threads - 1) / threads, static_cast<unsigned>(std::min<int64_t>(rows, 65535)));
    return cuda_status(launch_kernel(vec ? dequant8_kernel<T, true> : dequant8_kernel<T, false>, grid, dim3(threads), 0,
                                     static_cast<cudaStream_t>(stream), 1, codes, ldc, scale, static_cast<T*>(out), rows, h))
               ? W4A4_ERR_CUDA
               : ok();
  });
}

int w4a4_gemm8(const int8_t* a, int64_t lda, const float* sa, const int8_t* w, int64_t ldw, const float* sw,
               const void* bias, int32_t dtype, int64_t m, int32_t n, int32_t k, void* y, void* stream) {
  if (m < 0 || n <= 0 || k <= 0)
    return fail(W4A4_ERR_INVALID, "gemm8: invalid shape M=%lld N=%d K=%d", (long long)m, n, k);
  if (k >= 131072) return fail(W4A4_ERR_UNSUPPORTED, "gemm8: K must be below 131072 for exact int32 sums, got %d", k);
  if (m > 0x7fffff00LL) return fail(W4A4_ERR_UNSUPPORTED, "gemm8: too many rows: %lld", (long long)m);
  if (m == 0) return ok();
  if (!a || !sa || !w || !sw || !y) return fail(W4A4_ERR_INVALID, "gemm8: null pointer argument");
  if (lda < k || ldw < k) return fail(W4A4_ERR_INVALID, "gemm8: row stride below K = %d", k);
  if (!rows_aligned(a, lda, 1, 16) || !rows_aligned(w, ldw, 1, 16))
    return fail(W4A4_ERR_INVALID, "gemm8: rows of codes must begin at multiples of 16 bytes");
  if (!aligned(sw, 16)) return fail(W4A4_ERR_INVALID, "gemm8: channel scales must be 16-byte aligned");
  if (!aligned(y, 16) || (bias && !aligned(bias, 16)))
    return fail(W4A4_ERR_INVALID, "gemm8: y and bias must be 16-byte aligned");
  return launch_gemm8(a, lda, sa, w, ldw, sw, bias, dtype, m, n, k, y, static_cast<cudaStream_t>(stream));
}

int w4a4_gemm8_plan(int64_t m, int32_t n, int32_t k, const int32_t* clusters, int32_t* out) {
  if (m <= 0 || m > 0x7fffff00LL || n <= 0 || k <= 0 || k >= 131072 || !clusters || !out)
    return fail(W4A4_ERR_INVALID, "gemm8: invalid plan query");
  const int fit[4] = {clusters[0], clusters[1], clusters[2], clusters[3]};
  if (fit[0] < 2 || fit[1] < 1 || fit[2] < 0 || fit[3] < 0) return fail(W4A4_ERR_INVALID, "gemm8: invalid plan query");
  if (m <= kG8FewTokens) {
    const Gemm8FewPlan plan = gemm8_few_plan(m, n, k, fit[0]);
    out[0] = plan.deep ? W4A4_GEMM8_FEW_DEEP : plan.wide ? W4A4_GEMM8_FEW_WIDE : W4A4_GEMM8_FEW;
    out[1] = plan.half ? 8 : 16, out[2] = 1, out[3] = plan.ctas;
    return ok();
  }
  const Gemm8Plan plan = gemm8_plan(m, n, k, fit);
  out[0] = plan.pair ? W4A4_GEMM8_PAIR : W4A4_GEMM8_TILE;
  out[1] = plan.pair ? 256 : plan.tok_tile, out[2] = plan.split;
  out[3] = plan.pair ? 2 * std::min(fit[0] / 2, plan.n_tok_tiles * plan.n_w_tiles)
                     : plan.split * plan.n_tok_tiles * plan.n_w_tiles;
  return ok();
}

int w4a4_kv8_append(int8_t* k_codes, int8_t* v_codes, float* k_scale, float* v_scale, const int64_t* cache_stride,
                    int32_t capacity, const void* k, const int64_t* k_stride, const void* v, const int64_t* v_stride,
                    int32_t dtype, const uint8_t* valid, int64_t valid_stride, const int32_t* start, int32_t* lengths,
                    int32_t batch, int32_t tokens, int32_t heads, int32_t width, void* stream) {
  if (int e = check_cache8(k_codes, v_codes, k_scale, v_scale, cache_stride, batch, heads, width, capacity,
                           "kv8_append"))
    return e;
  if (tokens < 0) return fail(W4A4_ERR_INVALID, "kv8_append: invalid token count %d", tokens);
  if (tokens > 1 << 30) return fail(W4A4_ERR_UNSUPPORTED, "kv8_append: too many tokens: %d", tokens);
  if (batch == 0) return ok();
  if (!start || !lengths || !k_stride || !v_stride || (tokens > 0 && (!k || !v)))
    return fail(W4A4_ERR_INVALID, "kv8_append: null pointer argument");
  Kv8Params p{};
  p.codes[0] = k_codes, p.codes[1] = v_codes, p.scale[0] = k_scale, p.scale[1] = v_scale;
  p.x[0] = k, p.x[1] = v, p.start = start, p.valid = valid, p.valid_stride = valid_stride, p.lengths = lengths;
  p.cb = cache_stride[0], p.ct = cache_stride[1], p.ch = cache_stride[2];
  p.batch = batch, p.tokens = tokens, p.heads = heads, p.width = width, p.capacity = capacity;
  bool vec = true;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? v_stride : k_stride;
    p.xb[i] = s[0], p.xt[i] = s[1], p.xh[i] = s[2];
    vec = vec && aligned(p.x[i], 16) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
  }
  return by_dtype(dtype, false, "kv8_append", [&](auto tag) {
    using T = decltype(tag);
    // a run of `tokens` slots touches at most ceil((tokens - 1) / 16) + 1 blocks
    const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(tokens) + 14) / kKvBlock + 1),
                    static_cast<unsigned>(batch * heads));
    const auto kernel = vec ? kv8_append_kernel<T, true> : kv8_append_kernel<T, false>;
    return cuda_status(launch_kernel(kernel, grid, dim3(2 * width), 0, static_cast<cudaStream_t>(stream), 1, p))
               ? W4A4_ERR_CUDA
               : ok();
  });
}

int w4a4_kv8_values(const int8_t* k_codes, const int8_t* v_codes, const float* k_scale, const float* v_scale,
                    const int64_t* cache_stride, int32_t capacity, const int32_t* lengths, int32_t dtype, int32_t batch,
                    int32_t heads, int32_t width, void* k_out, void* v_out, void* stream) {
  if (int e = check_cache8(k_codes, v_codes, k_scale, v_scale, cache_stride, batch, heads, width, capacity,
                           "kv8_values"))
    return e;
  if (batch == 0) return ok();
  if (!lengths || !k_out || !v_out) return fail(W4A4_ERR_INVALID, "kv8_values: null pointer argument");
  if (!aligned(k_out, 16) || !aligned(v_out, 16))
    return fail(W4A4_ERR_INVALID, "kv8_values: outputs must be 16-byte aligned");
  Kv8ValuesParams p{};
  p.codes[0] = k_codes, p.codes[1] = v_codes, p.scale[0] = k_scale, p.scale[1] = v_scale;
  p.out[0] = k_out, p.out[1] = v_out, p.lengths = lengths;
  p.cb = cache_stride[0], p.ct = cache_stride[1], p.ch = cache_stride[2];
  p.batch = batch, p.heads = heads, p.width = width, p.capacity = capacity;
  return by_dtype(dtype, true, "kv8_values", [&](auto tag) {
    using T = decltype(tag);
    const dim3 grid(static_cast<unsigned>(capacity / kKvBlock), static_cast<unsigned>(batch * heads), 2);
    return cuda_status(launch_kernel(kv8_values_kernel<T>, grid, dim3(width), 0, static_cast<cudaStream_t>(stream), 1, p))
               ? W4A4_ERR_CUDA
               : ok();
  });
}

int w4a4_attention8_workspace(int32_t batch, int32_t tokens, int32_t q_heads, int32_t heads, int32_t width,
                              int32_t capacity, int64_t* bytes) {
  if (!bytes) return fail(W4A4_ERR_INVALID, "attention8: null pointer argument");
  if (batch < 0 || tokens < 0 || heads <= 0 || q_heads <= 0 || q_heads % heads || width <= 0 || capacity < 0)
    return fail(W4A4_ERR_INVALID, "attention8: invalid shape");
  *bytes = 0;
  if (batch == 0 || tokens == 0) return ok();
  int dev, fit[4];
  if (int e = current_device(&dev)) return e;
  if (int e = cluster_fit(dev, fit)) return e;
  const int64_t units = static_cast<int64_t>(batch) * heads, rows = static_cast<int64_t>(tokens) * (q_heads / heads);
  const Attn8Plan plan = attn8_plan(units, rows, capacity, width, fit);
  if (plan.splits > 1) *bytes = units * plan.splits * rows * (static_cast<int64_t>(width) * 4 + 8);
  return ok();
}

int w4a4_attention8(const void* q, const int64_t* q_stride, const int8_t* k_codes, const int8_t* v_codes,
                    const float* k_scale, const float* v_scale, const int64_t* cache_stride, int32_t capacity,
                    const int32_t* lengths, int32_t dtype, int32_t batch, int32_t tokens, int32_t q_heads, int32_t heads,
                    int32_t width, int32_t causal, float scale, void* out, void* workspace, int64_t workspace_bytes,
                    void* stream) {
  if (int e = check_cache8(k_codes, v_codes, k_scale, v_scale, cache_stride, batch, heads, width, capacity,
                           "attention8"))
    return e;
  if (dtype != W4A4_F16 && dtype != W4A4_BF16) return fail(W4A4_ERR_INVALID, "attention8: unsupported dtype code %d", dtype);
  if (tokens < 0 || q_heads <= 0 || q_heads % heads)
    return fail(W4A4_ERR_INVALID, "attention8: invalid tokens %d or %d query heads over %d heads", tokens, q_heads, heads);
  if (batch == 0 || tokens == 0) return ok();
  if (!q || !q_stride || !lengths || !out) return fail(W4A4_ERR_INVALID, "attention8: null pointer argument");
  if (!aligned(q, 16) || !aligned(out, 16) || q_stride[0] % 8 || q_stride[1] % 8 || q_stride[2] % 8)
    return fail(W4A4_ERR_INVALID, "attention8: query rows must begin at multiples of 16 bytes");
  if (static_cast<int64_t>(batch) * tokens * q_heads > 0x7fffffffLL)
    return fail(W4A4_ERR_UNSUPPORTED, "attention8: too many query rows");
  int dev, fit[4];
  if (int e = current_device(&dev)) return e;
  if (int e = cluster_fit(dev, fit)) return e;
  const int64_t units = static_cast<int64_t>(batch) * heads, rows = static_cast<int64_t>(tokens) * (q_heads / heads);
  const Attn8Plan plan = attn8_plan(units, rows, capacity, width, fit);
  Attn8Params p{};
  p.q = q, p.out = out, p.k = k_codes, p.v = v_codes, p.ks = k_scale, p.vs = v_scale, p.lengths = lengths;
  p.qb = q_stride[0], p.qt = q_stride[1], p.qh = q_stride[2];
  p.cb = cache_stride[0], p.ct = cache_stride[1], p.ch = cache_stride[2];
  p.tokens = tokens, p.heads = heads, p.group = q_heads / heads, p.capacity = capacity;
  p.rows = static_cast<int>(rows), p.splits = plan.splits;
  p.causal = causal != 0, p.scale = scale * 1.4426950408889634f, p.wait_limit_ns = g_wait_limit_ns.load();
  if (plan.splits > 1) {
    const int64_t parts = units * plan.splits * rows, need = parts * (static_cast<int64_t>(width) * 4 + 8);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < need)
      return fail(W4A4_ERR_INVALID, "attention8: needs a 16-byte aligned workspace of %lld bytes, got %lld", (long long)need,
                  (long long)(workspace ? workspace_bytes : 0));
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + parts * width);
  }
  return launch_attention8(p, plan, units, width, dtype, dev, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
