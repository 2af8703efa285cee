// The 4-bit K/V cache: rows of K and V into it and back.
//
// A value is decode(e2m1 code) * decode(e4m3 scale), one scale per 16 values along head_dim, by the rule that the framework's NVFP4
// operands use (quant_nvfp4_act_bf16 / fp4_encode, native/kernels/kernels.cu:222-277, tensor scale 1): 4.5 bits a value, a quarter of
// the bf16 cache and an eighth over. The product has at most six significant bits and lies in [2^-10, 2688], so a row read back is
// exact in bf16, and attention over the cache is attention over exactly those bf16 values.
//
// Both kernels move each byte once and do a few operations a value: bound by HBM (write: 2 bytes a bf16 value in, 0.5625 out). One
// thread handles one group of 16 of K and the same one of V, so that a warp's code words and scale bytes are contiguous and a thread has
// both of its loads in flight; the 32 bytes of a bf16 group go in one 256-bit access (as two of 16 bytes each store would touch 32
// sectors by half). 16384 rows of 4 heads of 256, there and back: 33.6 to 36.9 us for 172 MB (5.1 TB/s; 41.4 with 128-bit accesses and K and V in
// different threads); 64 scattered rows 4.2 us, both launches.
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

__device__ __forceinline__ void ld256(const void* p, uint32_t (&u)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
               : "l"(p));
}
__device__ __forceinline__ void st256(void* p, const uint32_t (&u)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]),
               "r"(u[7])
               : "memory");
}

// 16 consecutive values. ALIGN: 32-byte accesses, 16-byte ones, or one value at a time.
template <typename T, int ALIGN>
__device__ __forceinline__ void load16(const T* p, float (&f)[16]) {
  if constexpr (ALIGN == 1) {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = Ty<T>::ld(p + i);
  } else {
    constexpr int WORDS = 4 * (int)sizeof(T);
    uint32_t u[WORDS];
#pragma unroll
    for (int h = 0; h < WORDS; h += 8) {
      uint32_t q[8];
      if constexpr (ALIGN == 32) {
        ld256(reinterpret_cast<const uint32_t*>(p) + h, q);
      } else {
        const uint4 a = reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + h)[0], b = reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + h)[1];
        q[0] = a.x; q[1] = a.y; q[2] = a.z; q[3] = a.w; q[4] = b.x; q[5] = b.y; q[6] = b.z; q[7] = b.w;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) u[h + i] = q[i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = sizeof(T) == 4 ? __uint_as_float(u[i < WORDS ? i : 0]) : __uint_as_float(i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16);
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

// The cache row of token `row`, or -1: it is left out. I: an index type that holds rows * groups (divisions by the group count are
// most of what a thread computes beside its conversions).
__device__ __forceinline__ int64_t cache_row(const int64_t* slots, size_t row, size_t cache_rows, int* err) {
  const int64_t slot = slots ? slots[row] : (int64_t)row;
  if (slot >= 0 && (uint64_t)slot >= cache_rows) {
    set_err(err, DERR_CACHE_ROW);
    return -1;
  }
  return slot < 0 ? -1 : slot;
}

template <typename T, int ALIGN, typename I>
__global__ void __launch_bounds__(256) kv4_write_kernel(const T* __restrict__ k, size_t k_stride, const T* __restrict__ v, size_t v_stride,
                                                        const int64_t* __restrict__ slots, uint8_t* __restrict__ k_codes, uint8_t* __restrict__ k_scales,
                                                        uint8_t* __restrict__ v_codes, uint8_t* __restrict__ v_scales, size_t cache_rows, I total,
                                                        uint32_t groups, int* err) {
  const I i = (I)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const I row = i / groups;
  const uint32_t j = (uint32_t)(i - row * groups);
  const int64_t slot = cache_row(slots, row, cache_rows, err);
  if (slot < 0) return;
  float fk[16], fv[16];
  load16<T, ALIGN>(k + row * k_stride + (size_t)j * 16, fk);
  load16<T, ALIGN>(v + row * v_stride + (size_t)j * 16, fv);
  const size_t at = (size_t)slot * groups + j;
  uint2 codes;
  uint8_t scale;
  encode16<T>(fk, codes, scale);
  reinterpret_cast<uint2*>(k_codes)[at] = codes;
  k_scales[at] = scale;
  encode16<T>(fv, codes, scale);
  reinterpret_cast<uint2*>(v_codes)[at] = codes;
  v_scales[at] = scale;
}

// e2m1 * e4m3 is exact in f16, and in either output type. ALIGN: 32-byte stores, or 16-byte ones
template <typename T, int ALIGN>
__device__ __forceinline__ void decode16(const uint2 w, uint8_t scale, T* dst) {
  const __half_raw hr = __nv_cvt_fp8_to_halfraw(scale, __NV_E4M3);
  const __half2 s2 = __half2half2(*reinterpret_cast<const __half*>(&hr));
  uint32_t u[4 * sizeof(T)];
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const __half2_raw pr = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)((b < 4 ? w.x : w.y) >> (8 * (b & 3))), __NV_E2M1);
    const float2 p = __half22float2(__hmul2(*reinterpret_cast<const __half2*>(&pr), s2));
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(p.x, p.y);
      u[b] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      u[2 * b] = __float_as_uint(p.x);
      u[2 * b + 1] = __float_as_uint(p.y);
    }
  }
#pragma unroll
  for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = u[8 * h + i];
    if constexpr (ALIGN == 32) {
      st256(reinterpret_cast<uint32_t*>(dst) + 8 * h, q);
    } else {
      uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(dst) + 8 * h);
      d[0] = make_uint4(q[0], q[1], q[2], q[3]);
      d[1] = make_uint4(q[4], q[5], q[6], q[7]);
    }
  }
}

template <typename T, int ALIGN, typename I>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Cache c, size_t cache_rows, const int64_t* __restrict__ slots, T* __restrict__ k,
                                                       T* __restrict__ v, I total, uint32_t groups, int* err) {
  dependents_start();
  const I i = (I)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  size_t at = i;
  if (slots) {
    const I row = i / groups;
    const int64_t slot = cache_row(slots, row, cache_rows, err);
    if (slot < 0) return;
    at = (size_t)slot * groups + (size_t)(i - row * groups);
  }
  const uint2 wk = reinterpret_cast<const uint2*>(c.k.codes)[at], wv = reinterpret_cast<const uint2*>(c.v.codes)[at];
  const uint8_t sk = c.k.scales[at], sv = c.v.scales[at];
  decode16<T, ALIGN>(wk, sk, k + (size_t)i * 16);
  decode16<T, ALIGN>(wv, sv, v + (size_t)i * 16);
}

}  // namespace

template <typename T>
cudaError_t launch_kv4_write(const T* k, size_t k_stride, const T* v, size_t v_stride, const int64_t* slots, uint8_t* k_codes, uint8_t* k_scales,
                             uint8_t* v_codes, uint8_t* v_scales, size_t cache_rows, int rows, int kv, int hd, int* err, cudaStream_t s) {
  if (rows <= 0) return cudaSuccess;
  const uint32_t groups = (uint32_t)kv * (hd / 16);
  const size_t total = (size_t)rows * groups;
  const unsigned grid = (unsigned)((total + 255) / 256);
  auto at_steps = [&](size_t bytes) {  // rows and pointers on multiples of so many bytes
    return k_stride * sizeof(T) % bytes == 0 && v_stride * sizeof(T) % bytes == 0 && (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % bytes == 0;
  };
#define KV4_WRITE(ALIGN, I) \
  kv4_write_kernel<T, ALIGN, I><<<grid, 256, 0, s>>>(k, k_stride, v, v_stride, slots, k_codes, k_scales, v_codes, v_scales, cache_rows, (I)total, groups, err)
  if (total >= (1u << 31)) {
    if (at_steps(16)) KV4_WRITE(16, size_t);
    else KV4_WRITE(1, size_t);
  } else if (at_steps(32)) KV4_WRITE(32, uint32_t);
  else if (at_steps(16)) KV4_WRITE(16, uint32_t);
  else KV4_WRITE(1, uint32_t);
#undef KV4_WRITE
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_kv4_read(const Kv4Cache& c, size_t cache_rows, const int64_t* slots, T* k, T* v, int rows, int kv, int hd, int* err, cudaStream_t s) {
  if (rows <= 0) return cudaSuccess;
  const uint32_t groups = (uint32_t)kv * (hd / 16);
  const size_t total = (size_t)rows * groups;
  const unsigned grid = (unsigned)((total + 255) / 256);
  const bool wide = (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 32 == 0;
  if (total >= (1u << 31)) kv4_read_kernel<T, 16, size_t><<<grid, 256, 0, s>>>(c, cache_rows, slots, k, v, total, groups, err);
  else if (wide) kv4_read_kernel<T, 32, uint32_t><<<grid, 256, 0, s>>>(c, cache_rows, slots, k, v, (uint32_t)total, groups, err);
  else kv4_read_kernel<T, 16, uint32_t><<<grid, 256, 0, s>>>(c, cache_rows, slots, k, v, (uint32_t)total, groups, err);
  return cudaGetLastError();
}
#define INST_KV4(T)                                                                                                                                     \
  template cudaError_t launch_kv4_write<T>(const T*, size_t, const T*, size_t, const int64_t*, uint8_t*, uint8_t*, uint8_t*, uint8_t*, size_t, int, int, \
                                           int, int*, cudaStream_t);                                                                                    \
  template cudaError_t launch_kv4_read<T>(const Kv4Cache&, size_t, const int64_t*, T*, T*, int, int, int, int*, cudaStream_t);
INST_KV4(float)
INST_KV4(bf16)
