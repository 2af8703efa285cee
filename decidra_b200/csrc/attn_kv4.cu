// Attention over a K/V cache held in 4 bits (kv4.cu): one warp per (token, query head), keys one after the other with a running
// maximum and sum. The dot product is spread over the warp's lanes (head_dim / 32 values each).
#include "common.cuh"
#include "kv4.h"

namespace {

__device__ __forceinline__ float e4m3_value(uint8_t c) {
  const __half_raw hr = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&hr));
}

// D = head_dim / 32 values of one cache row and head, at dimension lane * D
template <int D>
__device__ __forceinline__ void cache_values(const Kv4Part& c, size_t row, int kv, int kh, int lane, float (&f)[D]) {
  const size_t at = row * kv + kh;
  const uint8_t* p = c.codes + at * (D * 16) + lane * (D / 2);
  const float s = e4m3_value(c.scales[at * (D * 2) + lane * D / 16]);
#pragma unroll
  for (int b = 0; b < D / 2; ++b) {
    const __half2_raw pr = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)p[b], __NV_E2M1);
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&pr));
    f[2 * b] = v.x * s;
    f[2 * b + 1] = v.y * s;
  }
}

template <int D>
struct Running {
  float m = -INFINITY, l = 0.f, o[D];
  __device__ __forceinline__ void add(const float (&q)[D], const float (&k)[D], const float (&v)[D], float scale) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < D; ++i) s += q[i] * k[i];
    s = warp_sum(s) * scale;
    const float n = fmaxf(m, s), a = expf(m - n), p = expf(s - n);
    m = n;
    l = l * a + p;
#pragma unroll
    for (int i = 0; i < D; ++i) o[i] = o[i] * a + p * v[i];
  }
};

// The sequence of a packed row: the last b with cu[b] <= t, or -1 behind the last sequence.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int B, int t) {
  if (t >= cu[B]) return -1;
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

template <int D>
__device__ __forceinline__ void store_row(const Running<D>& r, bf16* out, const bf16* gate, int lane) {
#pragma unroll
  for (int i = 0; i < D; ++i) {
    float o = r.l > 0.f ? r.o[i] / r.l : 0.f;
    if (gate) o *= sigmoid_f(__bfloat162float(gate[lane * D + i]));
    out[lane * D + i] = __float2bfloat16_rn(o);
  }
}

template <int D>
__global__ void __launch_bounds__(32) kv4_questions_kernel(const Kv4QuestionArgs a) {
  constexpr int HD = 32 * D;
  const int t = blockIdx.x, h = blockIdx.y, kh = h / (a.heads / a.kv), lane = threadIdx.x;
  const int b = sequence_of(a.cu, a.B, t);
  if (b < 0) return;
  const float scale = 1.0f / sqrtf((float)HD);
  float q[D], k[D], v[D];
  Running<D> r;
#pragma unroll
  for (int i = 0; i < D; ++i) {
    q[i] = __bfloat162float(a.q[t * a.q_stride + (size_t)h * HD + lane * D + i]);
    r.o[i] = 0.f;
  }
  for (int j = 0; j < a.n_state; ++j) {
    cache_values<D>(a.state.k, j, a.kv, kh, lane, k);
    cache_values<D>(a.state.v, j, a.kv, kh, lane, v);
    r.add(q, k, v, scale);
  }
  const int end = a.causal ? t + 1 : a.cu[b + 1];
  for (int j = a.cu[b]; j < end; ++j) {
#pragma unroll
    for (int i = 0; i < D; ++i) {
      k[i] = __bfloat162float(a.k_own[j * a.k_stride + (size_t)kh * HD + lane * D + i]);
      v[i] = __bfloat162float(a.v_own[j * a.v_stride + (size_t)kh * HD + lane * D + i]);
    }
    r.add(q, k, v, scale);
  }
  store_row<D>(r, a.out + ((size_t)t * a.heads + h) * HD, a.gate_qg ? a.gate_qg + t * a.qg_stride + (size_t)h * 2 * HD + HD : nullptr, lane);
}

}  // namespace

size_t kv4_question_workspace(int, int, int, int, int, int) { return 0; }
cudaError_t launch_kv4_questions(const Kv4QuestionArgs& a, void*, cudaStream_t s) {
  const dim3 grid(a.T, a.heads);
  if (a.hd == 64) kv4_questions_kernel<2><<<grid, 32, 0, s>>>(a);
  else if (a.hd == 128) kv4_questions_kernel<4><<<grid, 32, 0, s>>>(a);
  else kv4_questions_kernel<8><<<grid, 32, 0, s>>>(a);
  return cudaGetLastError();
}
