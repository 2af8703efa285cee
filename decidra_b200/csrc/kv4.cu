// The 4-bit K/V cache: rows of K and V into it and back.
//
// A value is decode(e2m1 code) * decode(e4m3 scale), one scale per 16 values along head_dim, by the rule that the framework's NVFP4
// operands use (quant_nvfp4_act_bf16 / fp4_encode, native/kernels/kernels.cu:222-277, tensor scale 1): 4.5 bits a value, a quarter of
// the bf16 cache and an eighth over. The product has at most six significant bits and lies in [2^-10, 2688], so a row read back is
// exact in bf16, and attention over the cache is attention over exactly those bf16 values.
//
// Both kernels move each byte once and do a few operations a value: bound by HBM (write: 2 bytes a bf16 value in, 0.5625 out). One
// thread handles one group of 16, so that a warp's loads, its code words and its scale bytes are each contiguous.
#include "common.cuh"
#include "kv4.h"

namespace {

__device__ __forceinline__ float e4m3_value(uint8_t c) {
  const __half_raw hr = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&hr));
}

// The rule of fp4_encode for any f32 quotient: the magnitude's index counts the borders it reaches (a tie goes up), the sign only for
// v < 0. A NaN reaches none.
__device__ __forceinline__ uint32_t e2m1_code(float x) {
  const float a = fabsf(x);
  const uint32_t m = (a >= 0.25f) + (a >= 0.75f) + (a >= 1.25f) + (a >= 1.75f) + (a >= 2.5f) + (a >= 3.5f) + (a >= 5.0f);
  return m | (x < 0.f ? 8u : 0u);
}

template <typename T, bool WIDE>
__device__ __forceinline__ void load16(const T* p, float (&f)[16]) {
  if constexpr (WIDE && sizeof(T) == 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[h];
      const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[8 * h + 2 * i] = __low2float(b[i]);
        f[8 * h + 2 * i + 1] = __high2float(b[i]);
      }
    }
  } else if constexpr (WIDE) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const float4 u = reinterpret_cast<const float4*>(p)[h];
      f[4 * h] = u.x; f[4 * h + 1] = u.y; f[4 * h + 2] = u.z; f[4 * h + 3] = u.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = Ty<T>::ld(p + i);
  }
}

template <typename T>
__device__ __forceinline__ void encode16(const float (&f)[16], uint2& codes, uint8_t& scale) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(f[i]));
  scale = (uint8_t)__nv_cvt_float_to_fp8(fmaxf(m / 6.0f, 1e-10f), __NV_SATFINITE, __NV_E4M3);
  const float sd = e4m3_value(scale);
  if constexpr (sizeof(T) == 2) {  // bf16 values: the conversion instruction gives the rule's codes (nvfp4_codes8)
    codes.x = nvfp4_codes8(&f[0], sd);
    codes.y = nvfp4_codes8(&f[8], sd);
  } else {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i >> 3] |= e2m1_code(f[i] / sd) << (4 * (i & 7));
    codes = make_uint2(w[0], w[1]);
  }
}

// blockIdx.y: 0 K, 1 V
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) kv4_write_kernel(const T* __restrict__ k, size_t k_stride, const T* __restrict__ v, size_t v_stride,
                                                        const int64_t* __restrict__ slots, uint8_t* __restrict__ k_codes, uint8_t* __restrict__ k_scales,
                                                        uint8_t* __restrict__ v_codes, uint8_t* __restrict__ v_scales, size_t cache_rows, size_t rows,
                                                        int groups, int* err) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * groups) return;
  const size_t row = i / (uint32_t)groups;
  const uint32_t j = (uint32_t)(i - row * groups);
  const int64_t slot = slots ? slots[row] : (int64_t)row;
  if (slot < 0) return;
  if ((uint64_t)slot >= cache_rows) {
    set_err(err, DERR_CACHE_ROW);
    return;
  }
  const bool second = blockIdx.y != 0;
  const T* src = (second ? v + row * v_stride : k + row * k_stride) + (size_t)j * 16;
  float f[16];
  load16<T, WIDE>(src, f);
  uint2 codes;
  uint8_t scale;
  encode16<T>(f, codes, scale);
  const size_t at = (size_t)slot * groups + j;
  reinterpret_cast<uint2*>(second ? v_codes : k_codes)[at] = codes;
  (second ? v_scales : k_scales)[at] = scale;
}

template <typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Cache c, size_t cache_rows, const int64_t* __restrict__ slots, T* __restrict__ k,
                                                       T* __restrict__ v, size_t rows, int groups, int* err) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * groups) return;
  const size_t row = i / (uint32_t)groups;
  const uint32_t j = (uint32_t)(i - row * groups);
  const int64_t slot = slots ? slots[row] : (int64_t)row;
  if (slot < 0) return;
  if ((uint64_t)slot >= cache_rows) {
    set_err(err, DERR_CACHE_ROW);
    return;
  }
  const Kv4Part part = blockIdx.y ? c.v : c.k;
  const size_t at = (size_t)slot * groups + j;
  const uint2 w = reinterpret_cast<const uint2*>(part.codes)[at];
  const __half_raw hr = __nv_cvt_fp8_to_halfraw(part.scales[at], __NV_E4M3);
  const __half2 s2 = __half2half2(*reinterpret_cast<const __half*>(&hr));
  T* dst = (blockIdx.y ? v : k) + i * 16;
  float f[16];
#pragma unroll
  for (int b = 0; b < 8; ++b) {  // e2m1 * e4m3 is exact in f16, and in either output type
    const __half2_raw pr = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)((b < 4 ? w.x : w.y) >> (8 * (b & 3))), __NV_E2M1);
    const float2 p = __half22float2(__hmul2(*reinterpret_cast<const __half2*>(&pr), s2));
    f[2 * b] = p.x;
    f[2 * b + 1] = p.y;
  }
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 u;
      __nv_bfloat162* b2 = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
      for (int n = 0; n < 4; ++n) b2[n] = __floats2bfloat162_rn(f[8 * h + 2 * n], f[8 * h + 2 * n + 1]);
      reinterpret_cast<uint4*>(dst)[h] = u;
    }
  } else {
#pragma unroll
    for (int h = 0; h < 4; ++h) reinterpret_cast<float4*>(dst)[h] = make_float4(f[4 * h], f[4 * h + 1], f[4 * h + 2], f[4 * h + 3]);
  }
}

}  // namespace

template <typename T>
cudaError_t launch_kv4_write(const T* k, size_t k_stride, const T* v, size_t v_stride, const int64_t* slots, uint8_t* k_codes, uint8_t* k_scales,
                             uint8_t* v_codes, uint8_t* v_scales, size_t cache_rows, int rows, int kv, int hd, int* err, cudaStream_t s) {
  if (rows <= 0) return cudaSuccess;
  constexpr int V = 16 / (int)sizeof(T);
  const int groups = kv * (hd / 16);
  const dim3 grid((unsigned)(((size_t)rows * groups + 255) / 256), 2);
  const bool wide = k_stride % V == 0 && v_stride % V == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0;
  (wide ? kv4_write_kernel<T, true> : kv4_write_kernel<T, false>)<<<grid, 256, 0, s>>>(k, k_stride, v, v_stride, slots, k_codes, k_scales, v_codes, v_scales,
                                                                                       cache_rows, (size_t)rows, groups, err);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_kv4_read(const Kv4Cache& c, size_t cache_rows, const int64_t* slots, T* k, T* v, int rows, int kv, int hd, int* err, cudaStream_t s) {
  if (rows <= 0) return cudaSuccess;
  const int groups = kv * (hd / 16);
  const dim3 grid((unsigned)(((size_t)rows * groups + 255) / 256), 2);
  kv4_read_kernel<T><<<grid, 256, 0, s>>>(c, cache_rows, slots, k, v, (size_t)rows, groups, err);
  return cudaGetLastError();
}
#define INST_KV4(T)                                                                                                                                     \
  template cudaError_t launch_kv4_write<T>(const T*, size_t, const T*, size_t, const int64_t*, uint8_t*, uint8_t*, uint8_t*, uint8_t*, size_t, int, int, \
                                           int, int*, cudaStream_t);                                                                                    \
  template cudaError_t launch_kv4_read<T>(const Kv4Cache&, size_t, const int64_t*, T*, T*, int, int, int, int*, cudaStream_t);
INST_KV4(float)
INST_KV4(bf16)
