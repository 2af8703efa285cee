// The 4-bit K/V cache (kv4.cu) and the attention over it (attn_kv4.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

// One of K or V: codes [rows, kv, hd / 2] (two e2m1 codes per byte, the even one in the low nibble), scales [rows, kv, hd / 16] (e4m3).
struct Kv4Part {
  const uint8_t* codes;
  const uint8_t* scales;
};
struct Kv4Cache {
  Kv4Part k, v;
};

// A kernel that may start while the one in front of it in the stream still runs: it does what needs nothing of that one, then waits for
// it (dependency_wait, in at least one thread of every block) and reads its results. The one in front lets it start with
// dependents_start; launched the ordinary way, either instruction does nothing.
#ifdef __CUDACC__
__device__ __forceinline__ void dependents_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, const A&... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = threads;
  c.dynamicSmemBytes = smem;
  c.stream = s;
  c.attrs = &at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}
#endif

inline bool kv4_head_dim_ok(int hd) { return hd == 64 || hd == 128 || hd == 256; }

// slots[i]: the cache row of token i (negative: the token is left out); null: row i.
template <typename T>
cudaError_t launch_kv4_write(const T* k, size_t k_stride, const T* v, size_t v_stride, const int64_t* slots, uint8_t* k_codes, uint8_t* k_scales,
                             uint8_t* v_codes, uint8_t* v_scales, size_t cache_rows, int rows, int kv, int hd, int* err, cudaStream_t s);
template <typename T>
cudaError_t launch_kv4_read(const Kv4Cache& c, size_t cache_rows, const int64_t* slots, T* k, T* v, int rows, int kv, int hd, int* err, cudaStream_t s);

// Packed questions over one shared state and their own keys (dcd_k_attention_kv4).
struct Kv4QuestionArgs {
  const __nv_bfloat16 *q, *k_own, *v_own, *gate_qg;
  size_t q_stride, k_stride, v_stride, qg_stride;
  Kv4Cache state;
  int n_state;
  __nv_bfloat16* out;
  const int32_t* cu;
  int B, T, heads, kv, hd, causal;
  int* err;
};
size_t kv4_question_workspace(int B, int T, int n_state, int heads, int kv, int hd);
cudaError_t launch_kv4_questions(const Kv4QuestionArgs& a, void* workspace, cudaStream_t s);

// The newest tokens of many sequences, each over its own rows of the cache (dcd_k_attention_kv4_decode).
struct Kv4DecodeArgs {
  const __nv_bfloat16 *q, *gate_qg;
  size_t q_stride, qg_stride;
  Kv4Cache cache;
  size_t cache_rows;
  const int64_t* seg_start;
  const int32_t* seg_len;
  int max_len;
  __nv_bfloat16* out;
  const int32_t* cu;
  int B, T, heads, kv, hd;
  int* err;
};
size_t kv4_decode_workspace(int B, int T, int max_len, int heads, int kv, int hd);
cudaError_t launch_kv4_decode(const Kv4DecodeArgs& a, void* workspace, cudaStream_t s);
