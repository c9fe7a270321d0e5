// KV cache rows: quantised to 8-bit floats as they are written, and read back.
//
// A row is the H values x of one (token, KV head).  Quantised (e4m3 code c and
// one exponent e per row):
//   e = clamp(ceil(log2(amax / 448)), -120, 119),  amax over the finite |x|
//   c = e4m3(x 2^-e)   round to nearest even, saturating at 448
//   value = c 2^e
// The scale is a power of two, so x 2^-e and c 2^e are exact and the 4-bit
// significand of e4m3 is the only rounding; c 2^e has 4 significant bits and is
// exact in bf16 (448 2^119 is its largest, 2^-129 its smallest).  A row of zeros has e = 0; an infinity saturates to 448 2^e;
// NaN stays NaN.  A bf16 cache takes the rows as they are.
//
// Both kernels are bound by memory: 8 values per lane (16-byte loads of bf16),
// H / 8 lanes per row with the row maximum by shuffles.
#include <cuda_fp8.h>
#include <torch/extension.h>

#include "../common/host.h"
#include "../common/sm100.cuh"
#include "checks.h"

namespace hb {
namespace {

struct RowStrides {   // in elements; the last dimension is contiguous
  long long b, s, n;
};

// One side (keys or values) of a write: source rows, cache rows, exponents.
struct WriteSide {
  const void* x;
  void* cache;
  int8_t* exps;
  RowStrides xs, cs, es;
};
struct WriteParams {
  WriteSide side[2];
  const int *starts, *counts;
  unsigned B, S, N;
  int C;
  int* status;
};

// 2^e, exact for -126 <= e <= 127.
HB_DEVICE float pow2i(int e) { return __int_as_float((e + 127) << 23); }

template <typename T>
HB_DEVICE void load8(const T* p, float (&f)[8]);
template <>
HB_DEVICE void load8(const __nv_bfloat16* p, float (&f)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <>
HB_DEVICE void load8(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// The row's exponent from its largest finite magnitude: amax = 1.m 2^x and
// 448 = 1.75 2^8, so the least e with amax <= 448 2^e is x - 8, or x - 7 when
// 1.m > 1.75.
HB_DEVICE int row_exponent(float amax) {
  if (amax == 0.f) return 0;
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -120), 119);
}

template <typename T, int H, bool QUANT>
__global__ void __launch_bounds__(256) kv_write_kernel(const WriteParams p) {
  constexpr int LPR = H / 8;   // lanes per row
  const WriteSide& sd = p.side[blockIdx.y];
  const unsigned row = (blockIdx.x * 256u + threadIdx.x) / LPR;
  const int l = threadIdx.x % LPR;
  const unsigned n = row % p.N, bs = row / p.N, i = bs % p.S, b = bs / p.S;
  bool on = b < p.B;
  long long at = 0;
  if (on) {
    on = p.counts == nullptr || (int)i < p.counts[b];
    at = (long long)p.starts[b] + i;
    if (on) on = index_ok(at, p.C, p.status);
  }
  float f[8] = {};
  if (on) load8<T>(reinterpret_cast<const T*>(sd.x) + b * sd.xs.b + i * sd.xs.s + n * sd.xs.n + l * 8, f);
  if constexpr (!QUANT) {
    if (!on) return;
    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(sd.cache) + b * sd.cs.b + at * sd.cs.s + n * sd.cs.n + l * 8;
    *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                                pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else {
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = fabsf(f[j]);
      if (a < INFINITY) amax = fmaxf(amax, a);   // false for NaN too
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!on) return;
    const int e = row_exponent(amax);
    const float inv = pow2i(-e);
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * h] * inv, f[4 * h + 1] * inv), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * h + 2] * inv, f[4 * h + 3] * inv), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | (hi << 16);
    }
    uint8_t* out = reinterpret_cast<uint8_t*>(sd.cache) + b * sd.cs.b + at * sd.cs.s + n * sd.cs.n + l * 8;
    *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
    if (l == 0) sd.exps[b * sd.es.b + at * sd.es.s + n * sd.es.n] = (int8_t)e;
  }
}

struct ReadSide {
  const void* cache;
  const int8_t* exps;
  __nv_bfloat16* out;   // [B, S, N, H] contiguous
  RowStrides cs, es;
};
struct ReadParams {
  ReadSide side[2];
  const int* starts;
  unsigned B, S, N;
  int C;
  int* status;
};

// fp8x4 -> two bf16x2 words, times 2^e (exact)
HB_DEVICE uint2 unpack4(uint32_t w, float sc) {
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
  const float2 x = __half22float2(__half2(a)), y = __half22float2(__half2(b));
  return make_uint2(pack_bf16x2(x.x * sc, x.y * sc), pack_bf16x2(y.x * sc, y.y * sc));
}

template <int H, bool QUANT>
__global__ void __launch_bounds__(256) kv_read_kernel(const ReadParams p) {
  constexpr int LPR = H / 8;
  const ReadSide& sd = p.side[blockIdx.y];
  const unsigned row = (blockIdx.x * 256u + threadIdx.x) / LPR;
  const int l = threadIdx.x % LPR;
  const unsigned n = row % p.N, bs = row / p.N, i = bs % p.S, b = bs / p.S;
  if (b >= p.B) return;
  const long long at = (p.starts ? (long long)p.starts[b] : 0) + i;
  uint4 o = make_uint4(0, 0, 0, 0);
  if (index_ok(at, p.C, p.status)) {
    const long long off = b * sd.cs.b + at * sd.cs.s + n * sd.cs.n + l * 8;
    if constexpr (QUANT) {
      const uint2 c = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(sd.cache) + off);
      const float sc = pow2i(sd.exps[b * sd.es.b + at * sd.es.s + n * sd.es.n]);
      const uint2 x = unpack4(c.x, sc), y = unpack4(c.y, sc);
      o = make_uint4(x.x, x.y, y.x, y.y);
    } else {
      o = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(sd.cache) + off);
    }
  }
  *reinterpret_cast<uint4*>(sd.out + ((long long)bs * p.N + n) * H + l * 8) = o;
}

RowStrides strides_of(const torch::Tensor& t) { return {t.stride(0), t.stride(1), t.stride(2)}; }

template <typename T, bool QUANT>
void launch_write(const WriteParams& p, int H, dim3 grid) {
  if (H == 32) kv_write_kernel<T, 32, QUANT><<<grid, 256, 0, cur_stream()>>>(p);
  else if (H == 64) kv_write_kernel<T, 64, QUANT><<<grid, 256, 0, cur_stream()>>>(p);
  else kv_write_kernel<T, 128, QUANT><<<grid, 256, 0, cur_stream()>>>(p);
}

dim3 rows_grid(int64_t rows, int64_t H) {
  const int64_t per = 256 / (H / 8), blocks = (rows + per - 1) / per;
  HB_CHECK(rows < (1ll << 31) && blocks < (1ll << 31), "kv_cache: too many rows for one call");
  return dim3((unsigned)blocks, 2, 1);
}

}  // namespace

// k, v [B, S, N, H] bf16 or fp32 into rows starts[b] + i (i < counts[b]) of the
// caches [B, C, N, H].
void kv_cache_write(torch::Tensor k_cache, torch::Tensor v_cache, OptTensor k_exp, OptTensor v_exp, torch::Tensor k,
                    torch::Tensor v, torch::Tensor starts, OptTensor counts) {
  const auto dev = k_cache.device();
  const c10::cuda::CUDAGuard guard(dev);
  check_cache(k_cache, v_cache, k_exp, v_exp, dev);
  const int64_t B = k_cache.size(0), N = k_cache.size(2), H = k_cache.size(3);
  need(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.device() == dev &&
           v.device() == dev && k.size(0) == B && k.size(2) == N && k.size(3) == H,
       "kv_cache_write: keys and values [B, S, N, H] of one type, shaped like the cache and on its device");
  need(k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kFloat, "kv_cache_write: bf16 or fp32 rows");
  need(!wants_grad(k) && !wants_grad(v), "kv_cache_write has no backward: call it under torch.no_grad()");
  const int64_t S = k.size(1);
  starts = whole(starts, B, dev, "kv_cache_write: starts, B whole numbers on the cache's device");
  if (counts) counts = whole(*counts, B, dev, "kv_cache_write: counts, B whole numbers on the cache's device");
  if (B * S * N == 0) return;
  k = aligned_rows(k), v = aligned_rows(v);
  const bool quant = k_exp.has_value();
  WriteParams p{};
  p.side[0] = {k.data_ptr(), k_cache.data_ptr(), quant ? k_exp->data_ptr<int8_t>() : nullptr, strides_of(k),
               strides_of(k_cache), quant ? strides_of(*k_exp) : RowStrides{}};
  p.side[1] = {v.data_ptr(), v_cache.data_ptr(), quant ? v_exp->data_ptr<int8_t>() : nullptr, strides_of(v),
               strides_of(v_cache), quant ? strides_of(*v_exp) : RowStrides{}};
  p.starts = starts.data_ptr<int>();
  p.counts = counts ? counts->data_ptr<int>() : nullptr;
  p.B = (unsigned)B, p.S = (unsigned)S, p.N = (unsigned)N, p.C = (int)k_cache.size(1);
  p.status = status_ptr();
  const dim3 grid = rows_grid(B * S * N, H);
  if (k.scalar_type() == at::kBFloat16) {
    if (quant) launch_write<__nv_bfloat16, true>(p, (int)H, grid);
    else launch_write<__nv_bfloat16, false>(p, (int)H, grid);
  } else {
    if (quant) launch_write<float, true>(p, (int)H, grid);
    else launch_write<float, false>(p, (int)H, grid);
  }
  HB_CUDA_CHECK(cudaGetLastError());
}

// Rows starts[b] .. starts[b] + S - 1 (from 0 without starts) of the caches as bf16 [B, S, N, H].
std::tuple<torch::Tensor, torch::Tensor> kv_cache_read(torch::Tensor k_cache, torch::Tensor v_cache, OptTensor k_exp,
                                                       OptTensor v_exp, OptTensor starts, int64_t S) {
  const auto dev = k_cache.device();
  const c10::cuda::CUDAGuard guard(dev);
  check_cache(k_cache, v_cache, k_exp, v_exp, dev);
  const int64_t B = k_cache.size(0), N = k_cache.size(2), H = k_cache.size(3);
  need(S >= 0, "kv_cache_read: n >= 0");
  if (starts) starts = whole(*starts, B, dev, "kv_cache_read: starts, B whole numbers on the cache's device");
  const auto opt = k_cache.options().dtype(at::kBFloat16);
  torch::Tensor k_out = torch::empty({B, S, N, H}, opt), v_out = torch::empty({B, S, N, H}, opt);
  if (B * S * N == 0) return {k_out, v_out};
  const bool quant = k_exp.has_value();
  ReadParams p{};
  p.side[0] = {k_cache.data_ptr(), quant ? k_exp->data_ptr<int8_t>() : nullptr, (__nv_bfloat16*)k_out.data_ptr(),
               strides_of(k_cache), quant ? strides_of(*k_exp) : RowStrides{}};
  p.side[1] = {v_cache.data_ptr(), quant ? v_exp->data_ptr<int8_t>() : nullptr, (__nv_bfloat16*)v_out.data_ptr(),
               strides_of(v_cache), quant ? strides_of(*v_exp) : RowStrides{}};
  p.starts = starts ? starts->data_ptr<int>() : nullptr;
  p.B = (unsigned)B, p.S = (unsigned)S, p.N = (unsigned)N, p.C = (int)k_cache.size(1);
  p.status = status_ptr();
  const dim3 grid = rows_grid(B * S * N, H);
  const cudaStream_t st = cur_stream();
  if (quant) {
    if (H == 32) kv_read_kernel<32, true><<<grid, 256, 0, st>>>(p);
    else if (H == 64) kv_read_kernel<64, true><<<grid, 256, 0, st>>>(p);
    else kv_read_kernel<128, true><<<grid, 256, 0, st>>>(p);
  } else {
    if (H == 32) kv_read_kernel<32, false><<<grid, 256, 0, st>>>(p);
    else if (H == 64) kv_read_kernel<64, false><<<grid, 256, 0, st>>>(p);
    else kv_read_kernel<128, false><<<grid, 256, 0, st>>>(p);
  }
  HB_CUDA_CHECK(cudaGetLastError());
  return {k_out, v_out};
}

}  // namespace hb
