// RMSNorm, with or without the residual's addition in front, whose output row goes straight to the operand format of the FP8 GEMM:
// e4m3 codes with one f32 scale per row (rmsnorm_bf16 / add_rmsnorm_bf16 followed by quant_fp8_per_token_bf16,
// native/kernels/kernels.cu:378-426, 182-205).
//
//   r = T(x + mix)                               (stored; the sum of squares and the output are taken from the stored value)
//   y = r * inv * (w + wofs),  inv = 1 / sqrt(mean(r^2) + eps)
//   s = max(max|y| * clip, 1e-10) / 448,  q = e4m3_satfinite(y / s)
//
// The two kernels it replaces move 2 bytes a value out and 2 (mostly from L2) in between them; here a row stays in registers from
// its one read to its one write, so the kernel is bound by its HBM bytes: x, mix and the residual in T, one byte out.
//
// Two forms of y. ROUND: y is rounded to T before it is quantised, which gives the bits of the two calls (the FP8 engine's results
// do not change), at the price of a second reduction, since the row's maximum is known only after inv. Without it y stays in f32 and
// is rounded to e4m3 only, and one reduction carries both sums: y = (r * (w + wofs)) * inv, rounding is monotone, so max|y| is
// max|r * (w + wofs)| * inv to the bit. The codes are e4m3((r * (w + wofs)) * (inv / scale)), one product a value where forming y and
// dividing it by the scale would be two: within three f32 roundings of y / scale, so that next to an e4m3 border a code may be the other one.
//
// The rounded form is a CTA per row: 6835 rows of 5120 bf16, as the engine calls it, 58 to 63 us (105 MB, 16 us at the copy rate; the two
// calls 71), 34 without the rounding.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace {

// V consecutive elements as f32: one 16-byte access, or one element where width, stride or address forbid it
template <typename T, int V> struct Pack;
template <> struct Pack<bf16, 8> {
  static __device__ __forceinline__ void ld(const bf16* p, float (&f)[8]) { unpack(*reinterpret_cast<const uint4*>(p), f); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __low2float(h[i]);
      f[2 * i + 1] = __high2float(h[i]);
    }
  }
  static __device__ __forceinline__ void st(bf16* p, const float (&f)[8]) {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = v;
  }
};
template <> struct Pack<float, 4> {
  static __device__ __forceinline__ void ld(const float* p, float (&f)[4]) { unpack(*reinterpret_cast<const uint4*>(p), f); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ void st(float* p, const float (&f)[4]) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};
template <typename T> struct Pack<T, 1> {
  static __device__ __forceinline__ void ld(const T* p, float (&f)[1]) { f[0] = Ty<T>::ld(p); }
  static __device__ __forceinline__ void st(T* p, const float (&f)[1]) { Ty<T>::st(p, f[0]); }
};

// The same V elements one by one, where the address forbids the access but their order is wanted
template <typename T, int V> struct Single {
  static __device__ __forceinline__ void ld(const T* p, float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = Ty<T>::ld(p + i);
  }
  static __device__ __forceinline__ void st(T* p, const float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) Ty<T>::st(p + i, f[i]);
  }
};

template <int V, bool WIDE = V != 1>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&f)[V]) {
  if constexpr (!WIDE) {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = (uint8_t)__nv_cvt_float_to_fp8(f[i], __NV_SATFINITE, __NV_E4M3);
  } else {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
             (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// Sum of a and maximum of b over the block; every thread gets both. `red` holds 64 floats.
__device__ __forceinline__ void block_sum_max(float& a, float& b, float* red) {
  a = warp_sum(a);
  b = warp_max(b);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (int)blockDim.x >> 5;
  if (lane == 0) { red[warp] = a; red[32 + warp] = b; }
  __syncthreads();
  a = warp_sum(lane < nw ? red[lane] : 0.f);
  b = warp_max(lane < nw ? red[32 + lane] : 0.f);
}

// One CTA per row, the row in registers: V * NV values a thread, cols <= V * NV * blockDim.x. x, mix and residual may be one buffer
// (every element is read before the same thread writes it), so none of them is restrict-qualified.
template <typename T, int V, int NV, bool ADD, bool ROUND, bool WIDE = true>
__global__ void __launch_bounds__(ROUND ? 256 : 1024) rmsnorm_fp8_kernel(const T* x, size_t x_stride, const T* mix, size_t mix_stride, const T* __restrict__ w,
                                                           T* residual, uint8_t* __restrict__ out, float* __restrict__ scales, int cols, float eps,
                                                           float wofs, float clip) {
  using P = std::conditional_t<WIDE, Pack<T, V>, Single<T, V>>;
  __shared__ float red[128];
  const size_t row = blockIdx.x;
  const int n = cols / V, nt = (int)blockDim.x;
  const T* xr = x + row * x_stride;
  float v[NV][V], m[ADD ? NV : 1][V], wv[ROUND ? 1 : NV][V];
  float ss = 0.f, mx = 0.f;
#pragma unroll
  for (int c = 0; c < NV; ++c) {  // all loads before the first use
    const int i = (int)threadIdx.x + c * nt;
    if (i < n) {
      P::ld(xr + (size_t)i * V, v[c]);
      if constexpr (ADD) P::ld(mix + row * mix_stride + (size_t)i * V, m[c]);
      if constexpr (!ROUND) P::ld(w + (size_t)i * V, wv[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int i = (int)threadIdx.x + c * nt;
    if (i < n) {
      if constexpr (ADD) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[c][j] = Ty<T>::rnd(v[c][j] + m[c][j]);
        P::st(residual + row * cols + (size_t)i * V, v[c]);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) ss += v[c][j] * v[c][j];
      if constexpr (!ROUND) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[c][j] *= wv[c][j] + wofs;
          mx = fmaxf(mx, fabsf(v[c][j]));
        }
      }
    }
  }
  block_sum_max(ss, mx, red);
  const float inv = 1.0f / sqrtf(ss / (float)cols + eps);
  if constexpr (ROUND) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int i = (int)threadIdx.x + c * nt;
      if (i < n) {
        P::ld(w + (size_t)i * V, wv[0]);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[c][j] = Ty<T>::rnd(v[c][j] * inv * (wv[0][j] + wofs));
          mx = fmaxf(mx, fabsf(v[c][j]));
        }
      }
    }
    float unused = 0.f;
    block_sum_max(unused, mx, red + 64);
  } else {
    mx *= inv;
  }
  const float scale = fmaxf(mx * clip, 1e-10f) / 448.f;
  if (threadIdx.x == 0) scales[row] = scale;
  const float f = inv / scale;
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int i = (int)threadIdx.x + c * nt;
    if (i < n) {
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = ROUND ? v[c][j] / scale : v[c][j] * f;
      store_codes<V, WIDE && V != 1>(out + row * cols + (size_t)i * V, y);
    }
  }
}

// Rows of one access a thread (cols <= V * blockDim.x), any number of them: a CTA takes every gridDim.x-th row, keeps its part of the
// weights, and has the next row's loads on their way while it reduces this one. 8883 rows of 5120 bf16 with the residual: 56 us (5.7 TB/s,
// 87 % of the measured copy; 58 to 63 call after call) with one wave of CTAs, 59 with half as many again, 58 with a CTA per row; and with a CTA per row 67 with
// two accesses a thread, 82 with four.
template <typename T, int V, bool ADD>
__global__ void __launch_bounds__(1024) rmsnorm_fp8_rows_kernel(const T* x, size_t x_stride, const T* mix, size_t mix_stride, const T* __restrict__ w,
                                                                T* residual, uint8_t* __restrict__ out, float* __restrict__ scales, int rows, int cols,
                                                                float eps, float wofs, float clip) {
  __shared__ float red[2][64];
  const size_t at = (size_t)threadIdx.x * V;
  const bool in = at < (size_t)cols;
  float wv[V];
#pragma unroll
  for (int j = 0; j < V; ++j) wv[j] = 0.f;
  uint4 nx = make_uint4(0, 0, 0, 0), nm = nx;  // as loaded: converting them would wait for them
  auto fetch = [&](int row) {
    if (in && row < rows) {
      nx = *reinterpret_cast<const uint4*>(x + row * x_stride + at);
      if constexpr (ADD) nm = *reinterpret_cast<const uint4*>(mix + row * mix_stride + at);
    }
  };
  fetch(blockIdx.x);
  if (in) {
    Pack<T, V>::ld(w + at, wv);
#pragma unroll
    for (int j = 0; j < V; ++j) wv[j] += wofs;
  }
  int set = 0;
  for (int row = blockIdx.x; row < rows; row += gridDim.x, set ^= 1) {
    float v[V], ss = 0.f, mx = 0.f;
    Pack<T, V>::unpack(nx, v);
    if constexpr (ADD) {
      float m[V];
      Pack<T, V>::unpack(nm, m);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = Ty<T>::rnd(v[j] + m[j]);
    }
    fetch(row + gridDim.x);
    if constexpr (ADD) {
      if (in) Pack<T, V>::st(residual + (size_t)row * cols + at, v);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      ss += v[j] * v[j];
      v[j] *= wv[j];
      mx = fmaxf(mx, fabsf(v[j]));
    }
    block_sum_max(ss, mx, red[set]);  // two sets: the next row's partial sums may come before the last warp has read these
    const float inv = 1.0f / sqrtf(ss / (float)cols + eps);
    const float scale = fmaxf(mx * inv * clip, 1e-10f) / 448.f;
    if (threadIdx.x == 0) scales[row] = scale;
    const float f = inv / scale;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] *= f;
    if (in) store_codes<V>(out + (size_t)row * cols + at, v);
  }
}

// Rows that do not fit in a block's registers: the same function in three passes over the row (from L2 after the first).
template <typename T, bool ADD, bool ROUND>
__global__ void __launch_bounds__(1024) rmsnorm_fp8_long_kernel(const T* x, size_t x_stride, const T* mix, size_t mix_stride, const T* __restrict__ w,
                                                                T* residual, uint8_t* __restrict__ out, float* __restrict__ scales, int cols, float eps,
                                                                float wofs, float clip) {
  __shared__ float red[128];
  const size_t row = blockIdx.x;
  const T* xr = x + row * x_stride;
  float ss = 0.f, mx = 0.f;
  for (int i = threadIdx.x; i < cols; i += blockDim.x) {
    float r = Ty<T>::ld(xr + i);
    if constexpr (ADD) {
      r = Ty<T>::rnd(r + Ty<T>::ld(mix + row * mix_stride + i));
      Ty<T>::st(residual + row * cols + i, r);
    }
    ss += r * r;
    if constexpr (!ROUND) mx = fmaxf(mx, fabsf(r * (Ty<T>::ld(w + i) + wofs)));
  }
  block_sum_max(ss, mx, red);
  const float inv = 1.0f / sqrtf(ss / (float)cols + eps);
  const T* src = ADD ? residual + row * cols : xr;
  if constexpr (ROUND) {
    for (int i = threadIdx.x; i < cols; i += blockDim.x) mx = fmaxf(mx, fabsf(Ty<T>::rnd(Ty<T>::ld(src + i) * inv * (Ty<T>::ld(w + i) + wofs))));
    float unused = 0.f;
    block_sum_max(unused, mx, red + 64);
  } else {
    mx *= inv;
  }
  const float scale = fmaxf(mx * clip, 1e-10f) / 448.f;
  if (threadIdx.x == 0) scales[row] = scale;
  const float f = inv / scale;
  for (int i = threadIdx.x; i < cols; i += blockDim.x) {
    const float r = Ty<T>::ld(src + i), wv = Ty<T>::ld(w + i) + wofs;
    const float y[1] = {ROUND ? Ty<T>::rnd(r * inv * wv) / scale : r * wv * f};
    store_codes<1>(out + row * cols + i, y);
  }
}

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return 148;
  return sms;
}

template <typename T, bool ADD, bool ROUND>
cudaError_t launch(const T* x, size_t xs, const T* mix, size_t ms, const T* w, T* res, uint8_t* out, float* scales, int rows, int cols, float eps,
                   float wofs, float clip, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  auto al = [](const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; };
  const bool wide = cols % V == 0 && xs % V == 0 && al(x, 16) && al(w, 16) && al(out, V) && (!ADD || (ms % V == 0 && al(mix, 16) && al(res, 16)));
  auto threads = [](int items, int per) { return ((items + per - 1) / per + 31) / 32 * 32; };
  if constexpr (ROUND) {
    // The summation order of the norm kernels whose bits it has to give (256 threads, f32 rows one element at a time). Warps that would have
    // nothing of a narrow row are left out: they add zeros (20000 rows of 256: with them 66 to 70 us, without 14, the two calls 60).
    if constexpr (sizeof(T) == 2) {
      if (cols % V == 0 && cols <= V * 4 * 256) {  // eight elements a thread, off 16 bytes too
        const int nt = min(256, threads(cols, V));
        if (wide) rmsnorm_fp8_kernel<T, V, 4, ADD, true><<<rows, nt, 0, s>>>(x, xs, mix, ms, w, res, out, scales, cols, eps, wofs, clip);
        else rmsnorm_fp8_kernel<T, V, 4, ADD, true, false><<<rows, nt, 0, s>>>(x, xs, mix, ms, w, res, out, scales, cols, eps, wofs, clip);
        return cudaGetLastError();
      }
    }
    if (cols <= 8 * 256) rmsnorm_fp8_kernel<T, 1, 8, ADD, true><<<rows, min(256, threads(cols, 1)), 0, s>>>(x, xs, mix, ms, w, res, out, scales, cols, eps, wofs, clip);
    else rmsnorm_fp8_long_kernel<T, ADD, true><<<rows, 256, 0, s>>>(x, xs, mix, ms, w, res, out, scales, cols, eps, wofs, clip);
  } else {
    if (wide && cols <= V * 1024 && rows <= 1 << 30) {  // the row number may pass `rows` by the grid
      const int nt = threads(cols / V, 1);
      const int sms = sm_count();
      int grid = rows, per_sm = 0;
      if (rows > sms) {  // one wave; how many CTAs that is depends on the form's registers (a question of 0.4 us on the host)
        CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, rmsnorm_fp8_rows_kernel<T, V, ADD>, nt, 0));
        grid = min(rows, sms * max(1, per_sm));
      }
      rmsnorm_fp8_rows_kernel<T, V, ADD><<<grid, nt, 0, s>>>(x, xs, mix, ms, w, res, out, scales, rows, cols, eps, wofs, clip);
    } else if (wide && cols <= V * 4 * 1024)
      rmsnorm_fp8_kernel<T, V, 4, ADD, false><<<rows, threads(cols / V, 4), 0, s>>>(x, xs, mix, ms, w, res, out, scales, cols, eps, wofs, clip);
    else if (!wide && cols <= 8 * 1024)
      rmsnorm_fp8_kernel<T, 1, 8, ADD, false><<<rows, threads(cols, 8), 0, s>>>(x, xs, mix, ms, w, res, out, scales, cols, eps, wofs, clip);
    else
      rmsnorm_fp8_long_kernel<T, ADD, false><<<rows, 1024, 0, s>>>(x, xs, mix, ms, w, res, out, scales, cols, eps, wofs, clip);
  }
  return cudaGetLastError();
}

}  // namespace

template <typename T>
cudaError_t launch_rmsnorm_fp8(const T* x, size_t x_stride, const T* mix, size_t mix_stride, const T* w, T* residual, uint8_t* out, float* scales, int rows,
                               int cols, float eps, bool zero_centered, float clip, bool round_t, cudaStream_t s) {
  if (rows <= 0) return cudaSuccess;
  const float wofs = zero_centered ? 1.0f : 0.0f;
  if (mix)
    return round_t ? launch<T, true, true>(x, x_stride, mix, mix_stride, w, residual, out, scales, rows, cols, eps, wofs, clip, s)
                   : launch<T, true, false>(x, x_stride, mix, mix_stride, w, residual, out, scales, rows, cols, eps, wofs, clip, s);
  return round_t ? launch<T, false, true>(x, x_stride, mix, mix_stride, w, residual, out, scales, rows, cols, eps, wofs, clip, s)
                 : launch<T, false, false>(x, x_stride, mix, mix_stride, w, residual, out, scales, rows, cols, eps, wofs, clip, s);
}
template cudaError_t launch_rmsnorm_fp8<float>(const float*, size_t, const float*, size_t, const float*, float*, uint8_t*, float*, int, int, float, bool,
                                               float, bool, cudaStream_t);
template cudaError_t launch_rmsnorm_fp8<bf16>(const bf16*, size_t, const bf16*, size_t, const bf16*, bf16*, uint8_t*, float*, int, int, float, bool, float,
                                              bool, cudaStream_t);
