// Attention of packed questions over one shared state held in 4 bits and their own bf16 keys, or causal attention over packed prompts
// (dcd_k_attention_kv4), on the sm_100a tensor cores.
//
// A state row is used by every tile of query rows, so it is decoded once per call: kv4_read writes the state's K and V as bf16 (exact)
// into the workspace, 2 x n_state x kv x head_dim x 2 bytes that mostly stay in L2, and the attention reads state and own keys alike
// through TMA.
//
// One CTA = (question, K/V head, tile of 128 / G tokens): the G query heads of a K/V head share its keys, so the 128 rows of an MMA
// tile are (token, head) pairs, brought in by a 3-D TMA box. Keys come in tiles of 128, the state's first, then the question's own:
//   S = Q K^T      tcgen05.mma, both operands from shared memory, S[j] in one of two 128-column TMEM buffers
//   P = softmax    of S[j]: one thread per row and two groups of four warps, one for even, one for odd tiles. While one group is in its
//                  exponentials the other is in the barriers, TMEM loads and stores around its own, so neither unit waits for a
//                  round trip, and no row is split between threads. Rescaling is lazy: O is rescaled only when a row's maximum has
//                  grown by more than 2^8; the groups hand the maximum in use from tile to tile through shared memory.
//   O += P V       P as the TMEM operand (over S[j]), V from shared memory, O in TMEM
// The tensor core runs S[0], S[1], then P.V[j], S[j + 2] in turn: a tile's softmax has a whole tile's products to hide behind.
// K and V come through one ring in the order in which they are used, so that the loads run two and more product phases ahead. A slot is
// 32 KB (16 KB at head_dim 64, a whole tile): with 16 KB slots the issuing warp, which spends 200 to 300 cycles on a slot beside its
// products (a satisfied wait alone takes 100 to 170), was slower than the tensor core: 4360 cycles a tile of 2048 at head_dim 256.
//
// Keys that do not exist are never multiplied as they lie in memory: the state's map ends at its last row (zeros behind it); of the own
// keys' last tile only steps of 16 with a key in them are multiplied, and the rows behind the last key are zeroed in shared memory
// first, so that whatever the next question holds there (NaN included) meets no product. A row's masked scores are replaced, not added to.
//
// Few CTAs over many keys leave SMs idle; the key tiles are then split over gridDim.z CTAs whose parts a second kernel adds up.
// All waits are bounded; one that gives up raises the error word, and the CTA drains and exits.
#include <cuda.h>

#include "common.cuh"
#include "gemm_tcgen05.h"
#include "kv4.h"
#include "tc_common.cuh"

namespace kvq {
using namespace tcc;

constexpr int KT = 128;                   // keys of a tile
constexpr int NUM_THREADS = 320, ISSUER = 8, LOADER = 9;
constexpr uint32_t S_COL = 256;           // TMEM: O from column 0, S at 256 and 384
constexpr float RESCALE = 8.0f;           // log2 units
constexpr uint32_t BAR_BYTES = 512, M_BYTES = 2 * 128 * 4;

template <int HD> struct Shape {
  static constexpr uint32_t SLOT = HD == 64 ? 16384 : 32768;  // bytes of a ring slot
  static constexpr int NKB = HD / 64;                         // 64-dim slabs of Q and K
  static constexpr int SLABS = SLOT / 16384;                  // slabs of a K slot
  static constexpr int KSUB = SLOT / (2 * HD);                // keys of a V slot
  static constexpr uint32_t Q_BYTES = 128 * HD * 2;
  static constexpr int SLOTS = HD == 256 ? 5 : HD == 128 ? 6 : 10;
  static constexpr uint32_t SMEM = Q_BYTES + SLOTS * SLOT + M_BYTES + BAR_BYTES + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Params {
  const int32_t* cu;
  int B, T, n_state, heads, kv;
  int G, sub, tokens;   // query rows per token of a tile; tiles of heads per K/V head; tokens per tile
  int causal;
  const bf16* gate_qg;
  size_t qg_stride;
  bf16* out;
  float scale_log2e;
  int* err;
  float* ws_o;     // gridDim.z > 1: unnormalised O [part][row block][row][HD], row block = blockIdx.y * gridDim.x + tile
  float2* ws_ml;   // (maximum in log2 units, sum)
};

struct Tile {
  int off, L, t0, ntok;  // the question's first packed row and length; the tile's first token and its tokens
};

// The question and tokens of tile `want`, counted from the last one when `reverse` (a causal prompt's late tiles are its longest, and
// start first). Offsets are clamped to the batch, so that bad ones cannot lead outside it. All threads of the block take part;
// `sums` holds 2 + blockDim.x / 32 ints. False: there is no such tile.
__device__ __forceinline__ bool find_tile(const Params& p, int want, bool reverse, int* sums, Tile& tile) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
  auto tiles_of = [&](int i, int& off, int& len) {
    off = len = 0;
    if (i >= p.B) return 0;
    off = p.cu[i];
    const int end = p.cu[i + 1];
    if (off < 0 || end < off || end > p.T) {
      set_err(p.err, DERR_OFFSETS);
      off = 0;
      return 0;
    }
    len = end - off;
    return (len + p.tokens - 1) / p.tokens;
  };
  if (reverse) {
    int mine = 0, off, len;
    for (int i = tid; i < p.B; i += nt) mine += tiles_of(i, off, len);
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    int total = 0;
    for (int i = 0; i < nw; ++i) total += sums[i];
    want = total - 1 - want;
    __syncthreads();
    if (want < 0) return false;
  }
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += nt) {
    int off, len;
    const int n = tiles_of(b0 + tid, off, len);
    int incl = n;
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    int before = base, all = base;
    for (int i = 0; i < nw; ++i) {
      if (i < warp) before += sums[i];
      all += sums[i];
    }
    __syncthreads();
    if (want < all) {
      before += incl - n;
      if (want >= before && want < before + n) {
        sums[0] = off;
        sums[1] = len;
        sums[2] = (want - before) * p.tokens;
      }
      __syncthreads();
      tile.off = __shfl_sync(0xffffffffu, sums[0], 0);  // uniform for the compiler too: what the issuing warps compute from it stays
      tile.L = __shfl_sync(0xffffffffu, sums[1], 0);    // on the uniform datapath (an MMA costs 60 to 75 cycles to issue otherwise, 21 so)
      tile.t0 = __shfl_sync(0xffffffffu, sums[2], 0);
      tile.ntok = min(p.tokens, tile.L - tile.t0);
      return true;
    }
    base = all;
  }
  return false;
}

// The key tiles of a CTA: tiles [lo, lo + n) of the state's followed by the own ones (causal: as far as the tile's last token).
struct Keys {
  int n_st, lo, n;
  __device__ __forceinline__ Keys(const Params& p, const Tile& t, int part, int parts) {
    n_st = (p.n_state + KT - 1) / KT;
    const int all = n_st + ((p.causal ? t.t0 + t.ntok : t.L) + KT - 1) / KT;
    const int per = (all + parts - 1) / parts;
    lo = part * per;
    n = max(0, min(all, lo + per) - lo);
  }
  __device__ __forceinline__ bool state(int j) const { return lo + j < n_st; }
  __device__ __forceinline__ int key0(int j) const { return (state(j) ? lo + j : lo + j - n_st) * KT; }
  // keys of tile j that some row of the CTA may see
  __device__ __forceinline__ int valid(int j, const Params& p, const Tile& t) const {
    return min(KT, (state(j) ? p.n_state : p.causal ? t.t0 + t.ntok : t.L) - key0(j));
  }
};

template <int HD>
__global__ void __launch_bounds__(NUM_THREADS, 1)
kv4_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKs, const __grid_constant__ CUtensorMap tmVs,
                     const __grid_constant__ CUtensorMap tmKo, const __grid_constant__ CUtensorMap tmVo, const Params p) {
  using D = Shape<HD>;
  constexpr int NKB = D::NKB, SLABS = D::SLABS, KSUB = D::KSUB, SLOTS = D::SLOTS;
  constexpr uint32_t SLOT = D::SLOT;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), pad = ((raw + 1023u) & ~1023u) - raw;
  uint8_t* smem = smem_raw + pad;
  const uint32_t q_base = raw + pad, ring = q_base + D::Q_BYTES;
  float* m_used = reinterpret_cast<float*>(smem + D::Q_BYTES + SLOTS * SLOT);  // [2][128] by tile parity
  float* l_part = reinterpret_cast<float*>(smem + D::Q_BYTES);                 // [2][128] by group, over the ring, after the last product
  uint8_t* bars_ptr = smem + D::Q_BYTES + SLOTS * SLOT + M_BYTES;
  const uint32_t bars = ring + SLOTS * SLOT + M_BYTES;
  // by tile parity: S done, P written, P.V done, maximum published. A parity wait is sound while the barrier is at most one phase
  // behind the waiter: with two barriers that is two tiles, and nobody runs two tiles ahead of P.V (S[j] comes behind P.V[j - 2]).
  const uint32_t bar_q = bars, bar_s = bars + 8, bar_p = bars + 24, bar_o = bars + 40, bar_m = bars + 56, bar_done = bars + 72, bar_l = bars + 80;
  const uint32_t full = bars + 96, empty = full + 8 * SLOTS;
  static_assert(96 + 16 * SLOTS + 64 <= BAR_BYTES, "barrier area");
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars_ptr + BAR_BYTES - 64);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars_ptr + BAR_BYTES - 60);
  int* sums = reinterpret_cast<int*>(bars_ptr + BAR_BYTES - 56);  // 12 ints

  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31;
  Tile tile;
  if (!find_tile(p, blockIdx.x, p.causal != 0, sums, tile)) return;
  const int G = p.G, hg = blockIdx.y, kh = hg / p.sub, head0 = kh * (p.heads / p.kv) + (hg - kh * p.sub) * G;
  const Keys keys(p, tile, blockIdx.z, gridDim.z);
  const int n_tiles = keys.n;
  const size_t block_lin = ((size_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  if (n_tiles == 0) {  // more parts than key tiles
    if (threadIdx.x < 128) p.ws_ml[block_lin * 128 + threadIdx.x] = make_float2(-INFINITY, 0.f);
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(bar_q, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_s + 8 * i, 1);
      mbar_init(bar_p + 8 * i, 128);
      mbar_init(bar_o + 8 * i, 1);
      mbar_init(bar_m + 8 * i, 128);
    }
    mbar_init(bar_done, 1);
    mbar_init(bar_l, 256);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // rows behind the last (token, head) pair are never written by TMA: zeros, so that they stay finite
  {
    const int row0 = p.tokens * G, nz = (128 - row0) * 8;
    for (int i = threadIdx.x; i < NKB * nz; i += NUM_THREADS) {
      const int kb = i / nz, c = i - kb * nz;
      *reinterpret_cast<uint4*>(smem + kb * 16384 + row0 * 128 + c * 16) = make_uint4(0, 0, 0, 0);
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_holder, 0);

  if (warp == LOADER) {
    // ---- Q, then K[0], K[1], V[0], K[2], V[1], K[3] ... through the ring: the order in which the issuer uses them ------------------
    const bool el = elect_one();
    if (el) {
      mbar_expect_tx(bar_q, (uint32_t)(NKB * p.tokens * G * 128));
#pragma unroll
      for (int c = 0; c < NKB; ++c) tma_load_3d(q_base + c * 16384, &tmQ, bar_q, c * 64, head0, tile.off + tile.t0);
    }
    bool ok = true;
    int slot = 0;
    uint32_t use = 0;  // rounds of the ring
    auto next_slot = [&]() {
      if (use > 0) ok = mbar_wait_warp(empty + 8 * slot, (use - 1) & 1, abort_flag);
      return ok;
    };
    auto advance = [&]() {
      if (++slot == SLOTS) { slot = 0; ++use; }
    };
    for (int i = 0; i < n_tiles + 2 && ok; ++i) {
      if (i >= 2) {
        const int j = i - 2;
        const bool st = keys.state(j);
        const int row = keys.key0(j) + (st ? 0 : tile.off), valid = keys.valid(j, p, tile);
        for (int s = 0; s * KSUB < valid && next_slot(); ++s) {
          if (el) {
            mbar_expect_tx(full + 8 * slot, SLOT);
#pragma unroll
            for (int c = 0; c < NKB; ++c) tma_load_2d(ring + slot * SLOT + c * (KSUB * 128), st ? &tmVs : &tmVo, full + 8 * slot, kh * HD + c * 64, row + s * KSUB);
          }
          advance();
        }
      }
      if (i < n_tiles) {
        const bool st = keys.state(i);
        const int row = keys.key0(i) + (st ? 0 : tile.off);
        for (int s = 0; s < NKB / SLABS && ok && next_slot(); ++s) {
          if (el) {
            mbar_expect_tx(full + 8 * slot, SLOT);
#pragma unroll
            for (int c = 0; c < SLABS; ++c) tma_load_2d(ring + slot * SLOT + c * 16384, st ? &tmKs : &tmKo, full + 8 * slot, kh * HD + (s * SLABS + c) * 64, row);
          }
          advance();
        }
      }
    }
  } else if (warp == ISSUER) {
    const bool el = elect_one();
    bool ok = mbar_wait_warp(bar_q, 0, abort_flag);
    int slot = 0;
    uint32_t use = 0;
    auto wait_slot = [&]() {
      ok = mbar_wait_warp(full + 8 * slot, use & 1, abort_flag);
      if (ok) tc_fence_after();
      return ok;
    };
    auto advance = [&]() {
      if (++slot == SLOTS) { slot = 0; ++use; }
    };
    for (int i = 0; i < n_tiles + 2 && ok; ++i) {
      if (i >= 2) {  // O += P[j] V[j]; P[j] lies over S[j]: 16 keys = 8 columns of bf16 pairs
        const int j = i - 2;
        if (!(ok = mbar_wait_warp(bar_p + 8 * (j & 1), (uint32_t)((j >> 1) & 1), abort_flag))) break;
        tc_fence_after();
        const int valid = keys.valid(j, p, tile);
        constexpr uint32_t idesc = umma_idesc(128, HD, 1);
        const uint32_t pj = tmem + S_COL + (j & 1) * KT;
        for (int s = 0; s * KSUB < valid && wait_slot(); ++s) {
          const int left = valid - s * KSUB;
          const uint64_t dv = umma_desc(ring + slot * SLOT, KSUB * 128, 1024);
          if (left >= KSUB) {
            if (el) {
#pragma unroll
              for (int k = 0; k < KSUB / 16; ++k) umma_f16_ts(tmem, pj + (s * (KSUB / 16) + k) * 8, dv + (uint64_t)(k * 128), idesc, (j | s | k) != 0 ? 1u : 0u);
              umma_commit_to(empty + 8 * slot);
            }
          } else {
            const int steps = (left + 15) >> 4;
            if (left & 15) {  // rows behind the last key of the step
              const int rows = steps * 16 - left;
              for (int z = lane; z < rows * NKB * 8; z += 32) {
                const int r = z / (NKB * 8), c = z - r * (NKB * 8);
                *reinterpret_cast<uint4*>(smem + D::Q_BYTES + slot * SLOT + (c >> 3) * (KSUB * 128) + (left + r) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
            }
            if (el) {
              for (int k = 0; k < steps; ++k) umma_f16_ts(tmem, pj + (s * (KSUB / 16) + k) * 8, dv + (uint64_t)(k * 128), idesc, (j | s | k) != 0 ? 1u : 0u);
              umma_commit_to(empty + 8 * slot);
            }
          }
          advance();
        }
        if (!ok) break;
        if (el) {
          umma_commit_to(bar_o + 8 * (j & 1));
          if (j + 1 == n_tiles) umma_commit_to(bar_done);
        }
      }
      if (i < n_tiles) {  // S[i]
        const int valid = keys.valid(i, p, tile);
        const uint32_t d = tmem + S_COL + (i & 1) * KT;
        // a partial tile: the columns that hold a key, rounded up to the instruction's 16
        const uint32_t idesc = valid == KT ? umma_idesc(128, KT, 0) : umma_idesc(128, 0, 0) | ((uint32_t)((valid + 15) >> 4) << 18);
        for (int s = 0; s < NKB / SLABS && wait_slot(); ++s) {
          if (el) {
#pragma unroll
            for (int c = 0; c < SLABS; ++c) {
              const uint64_t dq = umma_desc(q_base + (s * SLABS + c) * 16384, 16, 1024), dk = umma_desc(ring + slot * SLOT + c * 16384, 16, 1024);
#pragma unroll
              for (int k = 0; k < 4; ++k) umma_f16(d, dq + (uint64_t)(k * 2), dk + (uint64_t)(k * 2), idesc, (s | c | k) != 0 ? 1u : 0u);
            }
            umma_commit_to(empty + 8 * slot);
          }
          advance();
        }
        if (ok && el) umma_commit_to(bar_s + 8 * (i & 1));
      }
    }
  } else {
    // ---- softmax: group h takes the tiles of its parity; thread r of a group has row r ----------------------------------------------
    const int h = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + S_COL + h * KT;
    const int tok = tile.t0 + r / G;  // the row's token in its question
    float m = -INFINITY, l = 0.f;     // what this group's part of the denominator is relative to, and that part
    bool ok = true;
    for (int j = h; j < n_tiles && ok; j += 2) {
      const uint32_t ph = (uint32_t)((j >> 1) & 1);
      int lim = keys.valid(j, p, tile);
      if (p.causal && !keys.state(j)) lim = min(lim, tok + 1 - keys.key0(j));
      ok = __all_sync(0xffffffffu, mbar_wait(bar_s + 8 * h, ph, abort_flag));
      if (!ok) break;
      tc_fence_after();
      float x[KT];
#pragma unroll
      for (int i = 0; i < KT; i += 32) tmem_ld32(s_tmem + i, reinterpret_cast<uint32_t*>(x + i));
      tmem_ld_wait();
      if (__any_sync(0xffffffffu, lim < KT)) {
#pragma unroll
        for (int i = 0; i < KT; ++i) x[i] = i < lim ? x[i] : -INFINITY;
      }
      float t4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int i = 4; i < KT; ++i) t4[i & 3] = fmaxf(t4[i & 3], x[i]);
      const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * p.scale_log2e;
      // the maximum in use so far, from the other group's tile before this one
      float before = -INFINITY;
      if (j > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_m + 8 * (h ^ 1), (uint32_t)(((j - 1) >> 1) & 1), abort_flag));
        if (!ok) break;
        before = m_used[(h ^ 1) * 128 + r];
      }
      const float now = top > before + RESCALE ? top : before;
      m_used[h * 128 + r] = now;
      mbar_arrive(bar_m + 8 * h);
      if (j > 0 && __any_sync(0xffffffffu, now != before)) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_o + 8 * (h ^ 1), (uint32_t)(((j - 1) >> 1) & 1), abort_flag));  // O is at rest
        if (!ok) break;
        tc_fence_after();
        const float f = now != before ? ex2(before - now) : 1.0f;
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t v[32];
          tmem_ld32(tmem + lanes + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
          tmem_st32(tmem + lanes + c, v);
        }
        tmem_st_wait();
      }
      if (now != m) {
        l *= ex2(m - now);  // m = -inf: l is 0
        m = now;
      }
      const float neg = now == -INFINITY ? 0.f : -now;  // a row that has seen nothing: every weight 2^-inf
      float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float a = ex2(fmaf(x[half * 64 + 2 * i], p.scale_log2e, neg)), b = ex2(fmaf(x[half * 64 + 2 * i + 1], p.scale_log2e, neg));
          l4[(2 * i) & 3] += a;
          l4[(2 * i + 1) & 3] += b;
          w[i] = pack_bf16(a, b);
        }
        tmem_st32(s_tmem + half * 32, w);
      }
      l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(bar_p + 8 * h);
    }
    // ---- epilogue: either group takes half of the head's dimensions --------------------------------------------------------------
    const int last = (n_tiles - 1) & 1, tt = r / G, head = head0 + r - tt * G;
    const bool live = tt < tile.ntok;
    const size_t t = (size_t)tile.off + tile.t0 + tt;
    const bf16* gate = p.gate_qg && live && gridDim.z == 1 ? p.gate_qg + t * p.qg_stride + (size_t)(2 * head + 1) * HD + h * (HD / 2) : nullptr;
    uint4 gv[HD / 16];  // on their way while the last product runs
    if (gate) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) gv[i] = *reinterpret_cast<const uint4*>(gate + i * 8);
    }
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar_m + 8 * last, (uint32_t)(((n_tiles - 1) >> 1) & 1), abort_flag));
    float end_m = -INFINITY;
    if (ok) {
      end_m = m_used[last * 128 + r];
      ok = __all_sync(0xffffffffu, mbar_wait(bar_done, 0, abort_flag));
    }
    if (ok) {
      l_part[h * 128 + r] = m == -INFINITY ? 0.f : l * ex2(m - end_m);
      mbar_arrive(bar_l);
      ok = __all_sync(0xffffffffu, mbar_wait(bar_l, 0, abort_flag));
    }
    if (ok) {
      tc_fence_after();
      const float sum = l_part[r] + l_part[128 + r];
      if (gridDim.z > 1) {
        if (h == 0) p.ws_ml[block_lin * 128 + r] = make_float2(end_m, sum);
        float* dst = p.ws_o + (block_lin * 128 + r) * HD;
#pragma unroll 1
        for (int c = h * (HD / 2); c < (h + 1) * (HD / 2); c += 32) {
          uint32_t v[32];
          tmem_ld32(tmem + lanes + c, v);
          tmem_ld_wait();
          if (live) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
        }
      } else {
        const float inv = sum > 0.f ? 1.0f / sum : 0.f;
        bf16* dst = p.out + (t * p.heads + head) * HD + h * (HD / 2);
#pragma unroll
        for (int c = 0; c < HD / 2; c += 32) {
          uint32_t v[32];
          tmem_ld32(tmem + lanes + h * (HD / 2) + c, v);
          tmem_ld_wait();
          if (live) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float o[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] = __uint_as_float(v[i * 8 + k]) * inv;
              if (gate) {
                const __nv_bfloat162* g2 = reinterpret_cast<const __nv_bfloat162*>(&gv[c / 8 + i]);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  o[2 * k] *= __fdividef(1.0f, 1.0f + __expf(-__low2float(g2[k])));
                  o[2 * k + 1] *= __fdividef(1.0f, 1.0f + __expf(-__high2float(g2[k])));
                }
              }
              *reinterpret_cast<uint4*>(dst + c + i * 8) = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) set_err(p.err, DERR_ATTN_TIMEOUT);
#pragma unroll 1
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies in flight land
    __syncthreads();
  }
  if (warp == ISSUER) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// out = sum_z O_z 2^(m_z - M) / sum_z l_z 2^(m_z - M), gated: one warp per row; grid (tiles, heads' tiles, 128 / 4 rows)
template <int HD>
__global__ void __launch_bounds__(128) kv4_attention_merge_kernel(const Params p, int parts) {
  constexpr int PER = HD / 32;
  __shared__ int sums[8];
  Tile tile;
  if (!find_tile(p, blockIdx.x, p.causal != 0, sums, tile)) return;
  const int lane = threadIdx.x & 31, r = blockIdx.z * 4 + (threadIdx.x >> 5), G = p.G;
  if (r >= tile.ntok * G) return;
  const int hg = blockIdx.y, kh = hg / p.sub, tt = r / G;
  const int head = kh * (p.heads / p.kv) + (hg - kh * p.sub) * G + r - tt * G;
  const size_t step = (size_t)gridDim.y * gridDim.x * 128, row0 = ((size_t)hg * gridDim.x + blockIdx.x) * 128 + r;
  float M = -INFINITY;
  for (int z = lane; z < parts; z += 32) {
    const float2 x = p.ws_ml[z * step + row0];
    if (x.y > 0.f) M = fmaxf(M, x.x);
  }
  M = warp_max(M);
  float acc[PER], sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int z = 0; z < parts; ++z) {
    const float2 x = p.ws_ml[z * step + row0];
    if (!(x.y > 0.f)) continue;  // a part without keys, or one that this row sees nothing of: it may have written no O
    const float w = ex2(x.x - M);
    sum += w * x.y;
    const float* src = p.ws_o + (z * step + row0) * HD + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; i += 2) {
      const float2 v = *reinterpret_cast<const float2*>(src + i);
      acc[i] += w * v.x;
      acc[i + 1] += w * v.y;
    }
  }
  const size_t t = (size_t)tile.off + tile.t0 + tt;
  const float inv = sum > 0.f ? 1.0f / sum : 0.f;
  const bf16* gate = p.gate_qg ? p.gate_qg + t * p.qg_stride + (size_t)(2 * head + 1) * HD + lane * PER : nullptr;
  bf16* dst = p.out + (t * p.heads + head) * HD + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; i += 2) {
    float a = acc[i] * inv, b = acc[i + 1] * inv;
    if (gate) {
      const __nv_bfloat162 g2 = *reinterpret_cast<const __nv_bfloat162*>(gate + i);
      a *= sigmoid_f(__low2float(g2));
      b *= sigmoid_f(__high2float(g2));
    }
    *reinterpret_cast<__nv_bfloat162*>(dst + i) = __floats2bfloat162_rn(a, b);
  }
}

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return 148;
  return sms;
}

struct Plan {
  int G, sub, tokens, tiles, parts;
  size_t state_bytes, ml_bytes, o_bytes;
};
Plan plan_of(int B, int T, int n_state, int heads, int kv, int hd) {
  Plan p;
  const int group = heads / kv;
  p.G = group;
  while (p.G > 128 || group % p.G != 0) --p.G;  // the rows of one token fit a tile
  p.sub = group / p.G;
  p.tokens = 128 / p.G;
  p.tiles = (T + p.tokens - 1) / p.tokens + B;
  // split the keys where there is no CTA for every SM and the state is at least eight tiles long: about two CTAs per SM, at least
  // two key tiles per part
  const int ctas = p.tiles * kv * p.sub, st_tiles = (n_state + KT - 1) / KT, sms = sm_count();
  p.parts = 1;
  if (ctas <= sms && st_tiles >= 8) p.parts = max(1, min(min(2 * sms / ctas, st_tiles / 2), 128));
  p.state_bytes = (size_t)2 * n_state * kv * hd * 2;
  const size_t rows = p.parts > 1 ? (size_t)p.parts * ctas * 128 : 0;
  p.ml_bytes = rows * sizeof(float2);
  p.o_bytes = rows * hd * sizeof(float);
  return p;
}

template <int HD>
cudaError_t run(const Kv4QuestionArgs& a, const Plan& pl, uint8_t* ws, cudaStream_t s) {
  bf16* ks = (bf16*)ws;
  bf16* vs = ks + (size_t)a.n_state * a.kv * HD;
  Params p;
  p.cu = a.cu;
  p.B = a.B;
  p.T = a.T;
  p.n_state = a.n_state;
  p.heads = a.heads;
  p.kv = a.kv;
  p.G = pl.G;
  p.sub = pl.sub;
  p.tokens = pl.tokens;
  p.causal = a.causal;
  p.gate_qg = a.gate_qg;
  p.qg_stride = a.qg_stride;
  p.out = a.out;
  p.scale_log2e = (1.0f / sqrtf((float)HD)) * 1.4426950408889634f;
  p.err = a.err;
  p.ws_ml = (float2*)(ws + pl.state_bytes);
  p.ws_o = (float*)(ws + pl.state_bytes + pl.ml_bytes);
  const uint64_t width = (uint64_t)a.kv * HD;
  constexpr int KSUB = Shape<HD>::KSUB;
  TcTensorMap q, ko, vo, ksm, vsm;
  int bad = tc_make_tmap_3d(&q, a.q, HD, a.heads, a.T, HD, a.q_stride, pl.G, pl.tokens);
  bad |= tc_make_tmap_strided(&ko, a.k_own, a.T, width, a.k_stride, KT);
  bad |= tc_make_tmap_strided(&vo, a.v_own, a.T, width, a.v_stride, KSUB);
  if (a.n_state > 0) {
    bad |= tc_make_tmap_strided(&ksm, ks, a.n_state, width, width, KT);
    bad |= tc_make_tmap_strided(&vsm, vs, a.n_state, width, width, KSUB);
  } else {
    ksm = ko;
    vsm = vo;
  }
  if (bad) return cudaErrorInvalidValue;
  if (a.n_state > 0) CUDA_TRY(launch_kv4_read<bf16>(a.state, a.n_state, nullptr, ks, vs, a.n_state, a.kv, HD, nullptr, s));
  CUDA_TRY(cudaFuncSetAttribute(kv4_attention_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<HD>::SMEM));
  const dim3 grid(pl.tiles, a.kv * pl.sub, pl.parts);
  auto map = [](const TcTensorMap& m) -> const CUtensorMap& { return *reinterpret_cast<const CUtensorMap*>(&m); };
  kv4_attention_kernel<HD><<<grid, NUM_THREADS, Shape<HD>::SMEM, s>>>(map(q), map(ksm), map(vsm), map(ko), map(vo), p);
  CUDA_TRY(cudaGetLastError());
  if (pl.parts > 1) kv4_attention_merge_kernel<HD><<<dim3(pl.tiles, a.kv * pl.sub, 32), 128, 0, s>>>(p, pl.parts);
  return cudaGetLastError();
}

}  // namespace kvq

size_t kv4_question_workspace(int B, int T, int n_state, int heads, int kv, int hd) {
  const kvq::Plan p = kvq::plan_of(B, T, n_state, heads, kv, hd);
  return p.state_bytes + p.ml_bytes + p.o_bytes;
}

cudaError_t launch_kv4_questions(const Kv4QuestionArgs& a, void* workspace, cudaStream_t s) {
  const kvq::Plan p = kvq::plan_of(a.B, a.T, a.n_state, a.heads, a.kv, a.hd);
  if (a.kv * p.sub > 65535) return cudaErrorInvalidValue;
  if (a.hd == 256) return kvq::run<256>(a, p, (uint8_t*)workspace, s);
  if (a.hd == 128) return kvq::run<128>(a, p, (uint8_t*)workspace, s);
  return kvq::run<64>(a, p, (uint8_t*)workspace, s);
}
