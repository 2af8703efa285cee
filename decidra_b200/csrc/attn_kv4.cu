// Attention of packed questions over one shared state held in 4 bits and their own bf16 keys, or causal attention over packed prompts
// (dcd_k_attention_kv4), on the sm_100a tensor cores.
//
// A state row is used by every tile of query rows, so it is decoded once per call: kv4_read writes the state's K and V as bf16 (exact)
// into the workspace, 2 x n_state x kv x head_dim x 2 bytes that mostly stay in L2, and the attention reads state and own keys alike
// through TMA.
//
// A work item = (question, tile of 128 / G tokens, K/V head): the G query heads of a K/V head share its keys, so the 128 rows of an MMA
// tile are (token, head) pairs, brought in by a 3-D TMA box. One CTA per SM goes through its items one after the other; the loads and
// the first S products of an item run while the rows of the item before it are still being written. Keys come in tiles of 128, the
// state's first, then the question's own:
//   S = Q K^T      tcgen05.mma, both operands from shared memory, S[j] in one of the 128-column TMEM buffers
//   P = softmax    of S[j]: one thread per row and two groups of four warps, one for even, one for odd tiles. While one group is in its
//                  exponentials the other is in the barriers, TMEM loads and stores around its own, so neither unit waits for a
//                  round trip, and no row is split between threads. Rescaling is lazy: O is rescaled only when a row's maximum has
//                  grown by more than 2^8; the groups hand the maximum in use from tile to tile through shared memory.
//   O += P V       P as the TMEM operand (over S[j]), V from shared memory, O in TMEM. The weights enter it as bf16, as they do in the
//                  framework's bf16 attention (the operand has to be V's type): at most 2^-8 of each, independent of one another. Their sum is
//                  taken in f32 before that. Against 64 bits the output's rms error is 0.0020 to 0.0023 of it, where rounding it alone leaves 0.0016
// The tensor core runs S[0], S[1], then P.V[j], S[j + 2] in turn, so a tile's softmax has a whole tile's products to hide behind; up to
// head_dim 128 TMEM holds a third S, and a group finds its next scores there when it has written its weights (head_dim 128: 980 -> 885 ns
// a tile, 64: 965 -> 800). One warp issues both products: S[j + 2] overwrites P[j], and only one thread's products are sure to run in
// the order in which they were issued. K and V come through one ring of 32 KB slots (16 KB at head_dim 64, a whole tile) in the order in
// which they are used, so that the loads run two and more product phases ahead. A barrier wait that is already satisfied still takes 100
// to 170 cycles, which made the issuing warp slower than the tensor core (2048 cycles a tile at head_dim 256: 4360 with 16 KB slots, 3080
// with 32 KB), so another warp waits in its place (364 -> 330 us over 64 questions of about 107 tokens and 2048 state rows).
// The rows of O leave through a ring slot too: lane = row in TMEM, and sixteen bytes a row would be 32 lines a store; staged, a
// store covers four rows of 64 bytes.
//
// Keys that do not exist are never multiplied as they lie in memory: the state's map ends at its last row (zeros behind it); of the own
// keys' last tile only steps of 16 with a key in them are multiplied, and the rows behind the last key are zeroed in shared memory
// first, so that whatever the next question holds there (NaN included) meets no product. A row's masked scores are replaced, not added to.
//
// Few items over many keys leave SMs idle; the key tiles are then split into parts, items of their own, which a second kernel adds up.
//
// 64 questions of about 107 tokens over 2048 rows, 24 heads of 256, gated: 322 to 337 us (385 to 400 one after the other for 20 ms and more: the
// power limit), 1050 to 1090 TFLOP/s of the 1648 that a library product reaches;
// the tensor pipe is busy 56 % of the time, a tile takes 2400 to 2600 cycles for 2048 of products (S[j + 2] waits for P.V[j]), and a
// quarter of an item is its start, its masked tile and its rows. Five causal prompts of 1051 to 1814 tokens, 16 heads of 128: 67 to 83 us,
// bounded by the issue slots that the softmax and the issuing warp share.
// All waits are bounded; one that gives up raises the error word, and the CTA drains and exits.
#include <cuda.h>

#include "common.cuh"
#include "gemm_tcgen05.h"
#include "kv4.h"
#include "tc_common.cuh"

namespace kvq {
using namespace tcc;

constexpr int KT = 128;                   // keys of a tile
constexpr int NUM_THREADS = 352, ISSUER = 8, LOADER = 9, WAITER = 10;  // warps 0-7: softmax and epilogue
constexpr int MAX_ITEMS = 64;             // work items of a CTA
constexpr int EVENTS = 14;                // hardware barriers 1 to 14
constexpr float RESCALE = 8.0f;           // log2 units
constexpr uint32_t BAR_BYTES = 512, ROW_BYTES = 4 * 128 * 4, TABLE_BYTES = MAX_ITEMS * 8;

template <int HD> struct Shape {
  static constexpr uint32_t SLOT = HD == 64 ? 16384 : 32768;  // bytes of a ring slot
  static constexpr int NKB = HD / 64;                         // 64-dim slabs of Q and K
  static constexpr int SLABS = SLOT / 16384;                  // slabs of a K slot
  static constexpr int KSUB = SLOT / (2 * HD);                // keys of a V slot
  static constexpr uint32_t Q_BYTES = 128 * HD * 2;
  static constexpr int SLOTS = HD == 256 ? 5 : HD == 128 ? 6 : 10;
  static constexpr int KP = NKB / SLABS, VP = KT / KSUB;      // slots of a tile's K and V
  // TMEM: O from column 0, the S buffers behind it
  static constexpr int SB = HD == 256 ? 2 : 3;
  static constexpr uint32_t S_COL = HD == 256 ? 256 : 128;
  static constexpr uint32_t SMEM = Q_BYTES + SLOTS * SLOT + ROW_BYTES + BAR_BYTES + TABLE_BYTES;
  static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
  static_assert(SLOTS + SB < EVENTS, "events announced ahead");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// sigmoid with the hardware exponential and reciprocal (2 ulp or so in f32, 0 below 2^-126; the product is rounded to bf16). Split and whole
// questions share it
__device__ __forceinline__ float gate_of(float g) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(g * -1.4426950408889634f)));
  return r;
}

// Two f32 operations an instruction, each rounded as by itself: the softmax and the issuing warp share the issue slots (64 questions 336 -> 327 us,
// a tile at head_dim 128 877 -> 820 ns)
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
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
  int parts, max_tiles;
  float* ws_o;     // parts > 1: unnormalised O [part][heads' tile][token tile][row][HD]
  float2* ws_ml;   // (maximum in log2 units, sum)
};

struct Tile {
  int off, L, t0, ntok;  // the question's first packed row and length; the tile's first token and its tokens
};

// Token tiles of sequence i, its offset and length. Offsets that leave the batch count as an empty sequence.
__device__ __forceinline__ int tiles_of(const Params& p, int i, int& off, int& len) {
  off = p.cu[i];
  const int end = p.cu[i + 1];
  if (off < 0 || end < off || end > p.T) {
    set_err(p.err, DERR_OFFSETS);
    off = len = 0;
    return 0;
  }
  len = end - off;
  return (len + p.tokens - 1) / p.tokens;
}

// Calls found(sequence, its tiles before it, its tiles) for every sequence, each in one thread of the block, and returns the number of
// all tiles. `sums` holds an int per warp. Offsets that rise have at most max_tiles; where others add up to more, the sums stay at
// max_tiles + 1 (so that they cannot overflow), and the batch counts as empty.
template <typename F>
__device__ __forceinline__ int scan_tiles(const Params& p, int* sums, F found) {
  const int nt = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = nt >> 5, most = p.max_tiles + 1;
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += nt) {
    const int i = b0 + (int)threadIdx.x;
    int off, len;
    const int n = i < p.B ? min(tiles_of(p, i, off, len), most) : 0;
    int incl = n;
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl = min(incl + x, most);
    }
    if (lane == 31) sums[warp] = incl;
    const int up = __shfl_up_sync(0xffffffffu, incl, 1);
    __syncthreads();
    int before = base, all = base;
    for (int w = 0; w < nw; ++w) {
      if (w < warp) before = min(before + sums[w], most);
      all = min(all + sums[w], most);
    }
    __syncthreads();
    if (n > 0) found(i, lane > 0 ? min(before + up, most) : before, n);
    base = all;
  }
  if (base > p.max_tiles) {
    set_err(p.err, DERR_OFFSETS);
    return 0;
  }
  return base;
}

// The key tiles of a CTA: tiles [lo, lo + n) of the state's followed by the own ones (causal: as far as the tile's last token).
struct Keys {
  int n_st, lo, n;
  __device__ __forceinline__ Keys(const Params& p, const Tile& t, int part, int parts) {
    n_st = (p.n_state + KT - 1) / KT;
    const int all = n_st + ((p.causal ? t.t0 + t.ntok : t.L) + KT - 1) / KT;
    lo = 0;
    n = all;
    if (parts > 1) {  // a division of its own latency between two items
      const int per = (all + parts - 1) / parts;
      lo = part * per;
      n = max(0, min(all, lo + per) - lo);
    }
  }
  __device__ __forceinline__ bool state(int j) const { return lo + j < n_st; }
  __device__ __forceinline__ int key0(int j) const { return (state(j) ? lo + j : lo + j - n_st) * KT; }
  // keys of tile j that some row of the CTA may see
  __device__ __forceinline__ int valid(int j, const Params& p, const Tile& t) const {
    return min(KT, (state(j) ? p.n_state : p.causal ? t.t0 + t.ntok : t.L) - key0(j));
  }
};

__device__ __forceinline__ void named_sync(int id) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void named_arrive(int id) { asm volatile("barrier.cta.arrive %0, 64;" ::"r"(id) : "memory"); }

// Predicated instructions: a branch around each of a lane's rows costs more than the access
__device__ __forceinline__ uint2 ld_global_if(const void* p, bool there) {
  uint2 v;
  asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %3, 0;\nmov.b32 %0, 0;\nmov.b32 %1, 0;\n@q ld.global.v2.b32 {%0, %1}, [%2];\n}"
               : "=&r"(v.x), "=&r"(v.y)
               : "l"(p), "r"((int)there));
  return v;
}
__device__ __forceinline__ void st_global_if(void* p, uint2 v, bool there) {
  asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %3, 0;\n@q st.global.v2.b32 [%0], {%1, %2};\n}" ::"l"(p), "r"(v.x), "r"(v.y), "r"((int)there) : "memory");
}

// A causal prompt's late tiles are its longest and go first: sorted by where in their prompts they are, or, with more prompts than the
// lanes of a warp hold (by then a CTA has many items) or the keys split, from the batch's end. Sorted items go there and back again
// through the CTAs, so that the CTAs' sums stay close. Five prompts of 1051 to 1814 tokens, 16 heads of 128 over 2 K/V heads: from the
// end 91 to 94 us (the busiest SM has 58 key tiles, the mean is 43), sorted 72 to 83.
constexpr int SORTED = 4;  // prompts per lane
__device__ __forceinline__ bool sorted_items(const Params& p) { return p.causal && p.parts == 1 && p.B <= SORTED * 32; }
// The k-th item of a CTA. All in one direction otherwise: CTAs next to each other then stay closer in time and in what they read
// (64 questions, there and back: 338 us, one way 333).
__device__ __forceinline__ int item_of(const Params& p, int k) {
  const int c = (int)blockIdx.x, n = (int)gridDim.x;
  return k * n + (sorted_items(p) && (k & 1) ? n - 1 - c : c);
}
// The tile at place ti of the unsorted order
__device__ __forceinline__ int tile_of(const Params& p, int ti, int total) { return p.causal ? total - 1 - ti : ti; }

// What a work item is: its tokens, heads, part and keys. Every role goes through the same items; n_tiles == 0 (more parts than key tiles)
// leaves one out.
struct Item {
  Tile tile;
  int hg, kh, head0, z, ti;
  __device__ __forceinline__ Item(const Params& p, const int2* table, int k, int total) {
    const int nh = p.kv * p.sub, w = item_of(p, k), rest = w / nh;
    hg = w - rest * nh;
    z = ti = 0;  // only parts have a use for them
    if (p.parts > 1) {
      z = rest / total;
      ti = tile_of(p, rest - z * total, total);
    }
    // uniform for the compiler too, so that what the issuing warps compute from it stays on the uniform datapath
    const int b = __shfl_sync(0xffffffffu, table[k].x, 0);
    tile.t0 = __shfl_sync(0xffffffffu, table[k].y, 0);
    tile.off = p.cu[b];
    tile.L = p.cu[b + 1] - tile.off;
    tile.ntok = min(p.tokens, tile.L - tile.t0);
    kh = p.sub == 1 ? hg : hg / p.sub;
    head0 = kh * (p.heads / p.kv) + (hg - kh * p.sub) * p.G;
  }
};

template <int HD>
__global__ void __launch_bounds__(NUM_THREADS, 1)
kv4_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKs, const __grid_constant__ CUtensorMap tmVs,
                     const __grid_constant__ CUtensorMap tmKo, const __grid_constant__ CUtensorMap tmVo, const Params p) {
  using D = Shape<HD>;
  constexpr int NKB = D::NKB, SLABS = D::SLABS, KSUB = D::KSUB, SLOTS = D::SLOTS, KP = D::KP, VP = D::VP, SB = D::SB;
  constexpr uint32_t SLOT = D::SLOT, S_COL = D::S_COL;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t q_base = smem_u32(smem), ring = q_base + D::Q_BYTES;
  float* m_used = reinterpret_cast<float*>(smem + D::Q_BYTES + SLOTS * SLOT);  // [2][128] by tile parity
  float* l_part = m_used + 256;                                                // [2][128] by group
  uint8_t* bars_ptr = smem + D::Q_BYTES + SLOTS * SLOT + ROW_BYTES;
  int2* table = reinterpret_cast<int2*>(bars_ptr + BAR_BYTES);                 // (sequence, first token) of the CTA's items
  const uint32_t bars = ring + SLOTS * SLOT + ROW_BYTES;
  // by S buffer: S done, P written; by tile parity: P.V done, maximum published. Tiles are counted through all items of the CTA. A
  // parity wait is sound while the barrier is at most one phase behind the waiter: S[j + SB] comes behind P.V[j], P[j + SB] behind that,
  // and a tile's weights are written only after the maximum of the tile before it was read and that tile's P.V, if asked for, seen.
  // Once per item: Q loaded, Q no longer needed, last P.V done, sums exchanged, O read, the
  // epilogue's slot free.
  const uint32_t bar_s = bars, bar_p = bars + 24, bar_o = bars + 48, bar_m = bars + 64;
  const uint32_t bar_q = bars + 80, bar_q_free = bars + 88, bar_done = bars + 96, bar_l = bars + 104, bar_o_free = bars + 112, bar_e = bars + 120;
  const uint32_t full = bars + 128, empty = full + 8 * SLOTS;
  static_assert(128 + 16 * SLOTS + 64 <= BAR_BYTES, "barrier area");
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars_ptr + BAR_BYTES - 64);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars_ptr + BAR_BYTES - 60);
  int* sums = reinterpret_cast<int*>(bars_ptr + BAR_BYTES - 56);

  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31;
  if (q_base & 1023u) {  // the swizzled tiles need it; dynamic shared memory starts there as long as the kernel has no static
    if (threadIdx.x == 0) set_err(p.err, DERR_ATTN_TIMEOUT);
    dependency_wait();
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < SB; ++i) {
      mbar_init(bar_s + 8 * i, 1);
      mbar_init(bar_p + 8 * i, 128);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_o + 8 * i, 1);
      mbar_init(bar_m + 8 * i, 128);
    }
    mbar_init(bar_q, 1);
    mbar_init(bar_q_free, 1);
    mbar_init(bar_done, 1);
    mbar_init(bar_l, 256);
    mbar_init(bar_o_free, 256);
    mbar_init(bar_e, 256);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const int G = p.G;
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
  // the items: first the number of all tiles, then where each of this CTA's tiles lies
  int total = scan_tiles(p, sums, [](int, int, int) {});
  total = __shfl_sync(0xffffffffu, total, 0);
  const int nh = p.kv * p.sub, all_items = total * nh * p.parts;
  int n_items = all_items / (int)gridDim.x;
  if (item_of(p, n_items) < all_items) ++n_items;
  n_items = min(MAX_ITEMS, n_items);
  if (sorted_items(p)) {
    int n[SORTED];
#pragma unroll
    for (int q = 0; q < SORTED; ++q) {
      int off, len;
      n[q] = q * 32 + lane < p.B ? tiles_of(p, q * 32 + lane, off, len) : 0;
    }
    auto behind = [&](int i) {  // tiles with at least i others of their prompt in front of them
      int c = 0;
#pragma unroll
      for (int q = 0; q < SORTED; ++q) c += max(0, n[q] - i);
      return __reduce_add_sync(0xffffffffu, c);
    };
    for (int k = warp; k < n_items; k += NUM_THREADS / 32) {
      const int place = item_of(p, k) / nh;
      int i = 0, not_i = total;  // behind(i) > place >= behind(not_i)
      while (not_i - i > 1) {
        const int mid = (i + not_i) >> 1;
        if (behind(mid) > place) i = mid;
        else not_i = mid;
      }
      int before = place - behind(i + 1);  // prompts with such a tile in front of the one that is meant
#pragma unroll
      for (int q = 0; q < SORTED; ++q) {
        const uint32_t have = __ballot_sync(0xffffffffu, n[q] > i);
        if (n[q] > i && __popc(have & ((1u << lane) - 1u)) == before) table[k] = make_int2(q * 32 + lane, i * p.tokens);
        before -= __popc(have);
      }
    }
  } else {
    int* wanted = reinterpret_cast<int*>(l_part);  // the items' tile numbers; the rows' sums come here later
    if ((int)threadIdx.x < n_items) wanted[threadIdx.x] = tile_of(p, item_of(p, (int)threadIdx.x) / nh % total, total);
    __syncthreads();
    scan_tiles(p, sums, [&](int b, int before, int n) {
      for (int k = 0; k < n_items; ++k)
        if (wanted[k] >= before && wanted[k] < before + n) table[k] = make_int2(b, (wanted[k] - before) * p.tokens);
    });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_holder, 0);

  if (warp == LOADER) {
    // ---- per item Q, then K[0], K[1], V[0], K[2], V[1], K[3] ... through the ring: the order in which the issuer uses them; behind
    // the last V one slot for the epilogue --------------------------------------------------------------------------------------
    dependency_wait();  // the state's rows
    const bool el = elect_one();
    bool ok = true;
    int slot = 0, live = 0, e_slot = -1;
    uint32_t use = 0, e_parity = 0;  // use: rounds of the ring
    auto epilogue_done = [&]() {  // the slot that the epilogue of item live - 1 or the one before it was given
      if (ok && e_slot >= 0) ok = mbar_wait_warp(bar_e, e_parity, abort_flag);
      e_slot = -1;
    };
    auto next_slot = [&]() {
      if (use > 0) ok = mbar_wait_warp(empty + 8 * slot, (use - 1) & 1, abort_flag);
      if (slot == e_slot) epilogue_done();
      return ok;
    };
    auto advance = [&]() {
      if (++slot == SLOTS) { slot = 0; ++use; }
    };
    for (int k = 0; k < n_items && ok; ++k) {
      const Item it(p, table, k, total);
      const Keys keys(p, it.tile, it.z, p.parts);
      if (keys.n == 0) continue;
      if (live > 0 && !(ok = mbar_wait_warp(bar_q_free, (uint32_t)(live - 1) & 1, abort_flag))) break;
      if (el) {
        mbar_expect_tx(bar_q, (uint32_t)(NKB * p.tokens * G * 128));
#pragma unroll
        for (int c = 0; c < NKB; ++c) tma_load_3d(q_base + c * 16384, &tmQ, bar_q, c * 64, it.head0, it.tile.off + it.tile.t0);
      }
      for (int i = 0; i < keys.n + SB && ok; ++i) {
        if (i >= SB) {
          const bool st = keys.state(i - SB);
          const int row = keys.key0(i - SB) + (st ? 0 : it.tile.off);
          for (int s = 0; s < VP && next_slot(); ++s) {
            if (el) {
              mbar_expect_tx(full + 8 * slot, SLOT);
#pragma unroll
              for (int c = 0; c < NKB; ++c) tma_load_2d(ring + slot * SLOT + c * (KSUB * 128), st ? &tmVs : &tmVo, full + 8 * slot, it.kh * HD + c * 64, row + s * KSUB);
            }
            advance();
          }
        }
        if (i < keys.n) {
          const bool st = keys.state(i);
          const int row = keys.key0(i) + (st ? 0 : it.tile.off);
          for (int s = 0; s < KP && ok && next_slot(); ++s) {
            if (el) {
              mbar_expect_tx(full + 8 * slot, SLOT);
#pragma unroll
              for (int c = 0; c < SLABS; ++c) tma_load_2d(ring + slot * SLOT + c * 16384, st ? &tmKs : &tmKo, full + 8 * slot, it.kh * HD + (s * SLABS + c) * 64, row);
            }
            advance();
          }
        }
      }
      // The epilogue's slot is announced as full at once and, to keep its barriers in step, as empty too: what holds it is bar_e. One at
      // a time, so that bar_e is never two phases ahead of this warp.
      epilogue_done();
      if (!ok || !next_slot()) break;
      if (el) {
        mbar_arrive(full + 8 * slot);
        mbar_arrive(empty + 8 * slot);
      }
      e_slot = slot;
      e_parity = (uint32_t)live & 1;
      advance();
      ++live;
    }
  } else if (warp == WAITER) {
    // ---- waits for the issuer: the same barriers in the same order, each handed on through a hardware barrier. A satisfied mbarrier wait
    // takes 100 to 170 cycles, the hardware barrier 20 to 30; the tensor core's queue holds two or three products, so that what the
    // issuing warp waits is lost. V's slots are waited for in front of P, which comes last, and share its event. At most the ring's
    // slots and SB P are announced ahead, fewer than there are EVENTS. A wait that gave up is still announced, with the flag up, and
    // nothing after it ----------------------------------------------------------------------------------------------------------
    bool ok = true;
    int slot = 0, pb = 0;
    uint32_t use = 0, event = 0, pp = 0;  // pb, pp: buffer and phase of the next P
    auto wait = [&](uint32_t bar, uint32_t parity) { ok = ok && mbar_wait_warp(bar, parity, abort_flag); };
    auto wait_slot = [&]() {
      wait(full + 8 * slot, use & 1);
      if (++slot == SLOTS) { slot = 0; ++use; }
    };
    auto announce = [&]() { named_arrive(1 + (int)(event++ % EVENTS)); };
    for (int k = 0; k < n_items && ok; ++k) {
      const Item it(p, table, k, total);
      const Keys keys(p, it.tile, it.z, p.parts);
      if (keys.n == 0) continue;
      for (int i = 0; i < keys.n + SB && ok; ++i) {
        if (i >= SB) {
          for (int s = 0; s < VP; ++s) wait_slot();
          wait(bar_p + 8 * pb, pp);
          if (++pb == SB) { pb = 0; pp ^= 1; }
          announce();
        }
        if (i < keys.n) {
          for (int s = 0; s < KP && ok; ++s) {
            wait_slot();
            announce();
          }
        }
      }
      if (++slot == SLOTS) { slot = 0; ++use; }  // the epilogue's slot
    }
  } else if (warp == ISSUER) {
    const bool el = elect_one();
    bool ok = true;
    int slot = 0, live = 0, jj = 0, sb = 0, pb = 0;  // jj: tiles of the items before; sb, pb: buffers of the next S and P
    uint32_t event = 0;
    // What the waiter has seen. The flag is read here, in front of the products, and asked behind them: an event that was announced
    // after a wait had given up is the last, so that no other may be waited for
    auto next_event = [&]() {
      named_sync(1 + (int)(event++ % EVENTS));
      ok = *abort_flag == 0;
      tc_fence_after();
    };
    auto advance = [&]() { slot = slot + 1 == SLOTS ? 0 : slot + 1; };
    for (int k = 0; k < n_items && ok; ++k) {
      const Item it(p, table, k, total);
      const Keys keys(p, it.tile, it.z, p.parts);
      if (keys.n == 0) continue;
      if (!(ok = mbar_wait_warp(bar_q, (uint32_t)live & 1, abort_flag))) break;
      for (int i = 0; i < keys.n + SB && ok; ++i) {
        if (i >= SB) {  // O += P[j] V[j]; P[j] lies over S[j]: 16 keys = 8 columns of bf16 pairs
          const int j = i - SB, J = jj + j;
          next_event();  // V[j] and P[j]
          if (ok && j == 0 && live > 0) ok = mbar_wait_warp(bar_o_free, (uint32_t)(live - 1) & 1, abort_flag);  // O of the item before has been read
          if (!ok) break;  // the event may have been the last
          const int valid = keys.valid(j, p, it.tile);
          constexpr uint32_t idesc = umma_idesc(128, HD, 1);
          const uint32_t pj = tmem + S_COL + pb * KT;
          pb = pb + 1 == SB ? 0 : pb + 1;
          for (int s = 0; s < VP; ++s) {
            const int left = valid - s * KSUB;
            const uint64_t dv = umma_desc(ring + slot * SLOT, KSUB * 128, 1024);
            if (left >= KSUB) {
              if (el) {
#pragma unroll
                for (int x = 0; x < KSUB / 16; ++x) umma_f16_ts(tmem, pj + (s * (KSUB / 16) + x) * 8, dv + (uint64_t)(x * 128), idesc, (j | s | x) != 0 ? 1u : 0u);
                umma_commit_to(empty + 8 * slot);
              }
            } else {
              const int steps = max(0, (left + 15) >> 4);
              if (left > 0 && (left & 15)) {  // rows behind the last key of the step
                const int rows = steps * 16 - left;
                for (int z = lane; z < rows * NKB * 8; z += 32) {
                  const int r = z / (NKB * 8), c = z - r * (NKB * 8);
                  *reinterpret_cast<uint4*>(smem + D::Q_BYTES + slot * SLOT + (c >> 3) * (KSUB * 128) + (left + r) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
              }
              if (el) {
                for (int x = 0; x < steps; ++x) umma_f16_ts(tmem, pj + (s * (KSUB / 16) + x) * 8, dv + (uint64_t)(x * 128), idesc, (j | s | x) != 0 ? 1u : 0u);
                umma_commit_to(empty + 8 * slot);
              }
            }
            advance();
          }
          if (!ok) break;
          if (el) {
            umma_commit_to(bar_o + 8 * (J & 1));
            if (j + 1 == keys.n) umma_commit_to(bar_done);
          }
        }
        if (i < keys.n) {  // S[i]
          const int valid = keys.valid(i, p, it.tile);
          const uint32_t d = tmem + S_COL + sb * KT, done = bar_s + 8 * sb;
          sb = sb + 1 == SB ? 0 : sb + 1;
          // a partial tile: the columns that hold a key, rounded up to the instruction's 16
          const uint32_t idesc = valid == KT ? umma_idesc(128, KT, 0) : umma_idesc(128, 0, 0) | ((uint32_t)((valid + 15) >> 4) << 18);
          for (int s = 0; s < KP; ++s) {
            next_event();
            if (el) {
#pragma unroll
              for (int c = 0; c < SLABS; ++c) {
                const uint64_t dq = umma_desc(q_base + (s * SLABS + c) * 16384, 16, 1024), dk = umma_desc(ring + slot * SLOT + c * 16384, 16, 1024);
#pragma unroll
                for (int x = 0; x < 4; ++x) umma_f16(d, dq + (uint64_t)(x * 2), dk + (uint64_t)(x * 2), idesc, (s | c | x) != 0 ? 1u : 0u);
              }
              umma_commit_to(empty + 8 * slot);
            }
            advance();
            if (!ok) break;
          }
          if (!ok) break;
          if (el) {
            umma_commit_to(done);
            if (i + 1 == keys.n) umma_commit_to(bar_q_free);
          }
        }
      }
      advance();  // the epilogue's slot
      jj += keys.n;
      ++live;
    }
  } else {
    // ---- softmax: group h takes the tiles of its parity; thread r of a group has row r ----------------------------------------------
    const int h = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_tmem0 = tmem + lanes + S_COL;
    const int tt = r / G;  // the row's token in the tile
    bool ok = true;
    int live = 0, jj = 0;
    uint32_t slots_used = 0;
    for (int k = 0; k < n_items && ok; ++k) {
    const Item it(p, table, k, total);
    const Tile& tile = it.tile;
    const Keys keys(p, tile, it.z, p.parts);
    const int n_tiles = keys.n;
    const size_t block_lin = ((size_t)it.z * nh + it.hg) * p.max_tiles + it.ti;
    if (n_tiles == 0) {  // more parts than key tiles
      if (h == 0) p.ws_ml[block_lin * 128 + r] = make_float2(-INFINITY, 0.f);
      continue;
    }
    const int tok = tile.t0 + tt;  // ... and in its question
    if (p.gate_qg && p.parts == 1 && tt < tile.ntok) {  // the item's gates come to L2 now: all CTAs reach their epilogues at about the same time
      const bf16* gate = p.gate_qg + ((size_t)tile.off + tok) * p.qg_stride + (size_t)(2 * (it.head0 + r - tt * G) + 1) * HD + h * (HD / 2);
#pragma unroll
      for (int i = 0; i < HD / 2; i += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(gate + i));
    }
    float m = -INFINITY, l = 0.f;  // what this group's part of the denominator is relative to, and that part
    for (int j = (h ^ jj) & 1; j < n_tiles && ok; j += 2) {
      const uint32_t J = (uint32_t)(jj + j), ph_before = ((J - 1) >> 1) & 1, b = SB == 2 ? (uint32_t)h : J % SB;
      const uint32_t s_tmem = s_tmem0 + b * KT;
      int lim = keys.valid(j, p, tile);
      if (p.causal && !keys.state(j)) lim = min(lim, tok + 1 - keys.key0(j));
      // the maximum in use so far, from the other group's tile before this one: published long before S[j] is there
      float before = -INFINITY;
      if (j > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_m + 8 * (h ^ 1), ph_before, abort_flag));
        if (!ok) break;
        before = m_used[(h ^ 1) * 128 + r];
      }
      ok = __all_sync(0xffffffffu, mbar_wait(bar_s + 8 * b, SB == 2 ? (J >> 1) & 1 : (J / SB) & 1, abort_flag));
      if (!ok) break;
      tc_fence_after();
      // The scores are read from TMEM twice, 64 at a time, once for the maximum and once for the weights: a thread that keeps all 128 has
      // none of its registers left, and the straight code for them evicts the issuing warp's from the instruction cache (419 -> 364 us
      // over 64 questions of about 107 tokens and 2048 keys).
      // Keys that no row of the warp sees are left out 64 at a time, and only where some row sees some are they masked one by one.
      const int all_see = __reduce_min_sync(0xffffffffu, lim), some_see = __reduce_max_sync(0xffffffffu, lim);
      float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
      for (int c = 0; c < KT && c < some_see; c += 64) {
        float x[64];
#pragma unroll
        for (int i = 0; i < 64; i += 32) tmem_ld32(s_tmem + c + i, reinterpret_cast<uint32_t*>(x + i));
        tmem_ld_wait();
        if (all_see < c + 64) {
#pragma unroll
          for (int i = 0; i < 64; ++i) x[i] = c + i < lim ? x[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 64; ++i) t4[i & 3] = fmaxf(t4[i & 3], x[i]);
      }
      const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * p.scale_log2e;
      const float now = top > before + RESCALE ? top : before;
      m_used[h * 128 + r] = now;
      mbar_arrive(bar_m + 8 * h);
      if (j > 0 && __any_sync(0xffffffffu, now != before)) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_o + 8 * (h ^ 1), ph_before, abort_flag));  // O is at rest
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
      const float2 scale2 = make_float2(p.scale_log2e, p.scale_log2e), neg2 = make_float2(neg, neg);
      float2 l2[2] = {};
#pragma unroll 1
      for (int c = 0; c < KT; c += 64) {
        uint32_t w[32];
        if (c >= some_see) {
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = 0u;
          tmem_st32(s_tmem + c / 2, w);
          continue;
        }
        float x[64];
#pragma unroll
        for (int i = 0; i < 64; i += 32) tmem_ld32(s_tmem + c + i, reinterpret_cast<uint32_t*>(x + i));
        tmem_ld_wait();
        if (all_see < c + 64) {
#pragma unroll
          for (int i = 0; i < 64; ++i) x[i] = c + i < lim ? x[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float2 e = fma2(make_float2(x[2 * i], x[2 * i + 1]), scale2, neg2);
          e = make_float2(ex2(e.x), ex2(e.y));
          l2[i & 1] = add2(l2[i & 1], e);
          w[i] = pack_bf16(e.x, e.y);
        }
        tmem_st32(s_tmem + c / 2, w);
      }
      l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(bar_p + 8 * b);
    }
    // ---- epilogue: either group takes half of the head's dimensions, each warp its 32 rows, CH dimensions at a time: from TMEM (lane =
    // row) to the warp's part of the epilogue's slot, and from there in whole rows ---------------------------------------------------
    constexpr int CH = SLOT / 1024, LPR = CH / 4, RPP = 32 / LPR, PASSES = 32 / RPP;  // lanes per row, rows per pass
    const int last_j = jj + n_tiles - 1, last = last_j & 1;
    slots_used += (uint32_t)n_tiles * (KP + VP);
    const int e_slot = (int)(slots_used % SLOTS);
    const uint32_t e_phase = (slots_used / SLOTS) & 1;
    ++slots_used;
    // a lane's rows, four dimensions of each: where they go, and the gates of the first dimensions, on their way under the last product
    const int my_row = lane / LPR, my_c = lane % LPR;
    const float inv_g = 1.0f / (float)G;
    const bf16* gate0 = p.parts == 1 && p.gate_qg ? p.gate_qg + ((size_t)tile.off + tile.t0) * p.qg_stride + (size_t)(2 * it.head0 + 1) * HD + h * (HD / 2) + my_c * 4 : nullptr;
    bf16* out0 = p.out + (((size_t)tile.off + tile.t0) * p.heads + it.head0) * HD + h * (HD / 2) + my_c * 4;
    uint32_t gate_at[PASSES], out_at[PASSES];  // offsets of the rows; ~0: not a row of the question
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int R = (warp & 3) * 32 + ps * RPP + my_row, rt = (int)(((float)R + 0.5f) * inv_g);  // R / G, exact below 128
      const bool there = rt < tile.ntok;
      gate_at[ps] = (uint32_t)rt * (uint32_t)p.qg_stride + (uint32_t)(2 * (R - rt * G)) * HD;
      out_at[ps] = there ? (uint32_t)(rt * p.heads + R - rt * G) * HD : ~0u;
    }
    uint2 gv[PASSES];
    auto load_gates = [&](int c) {
#pragma unroll
      for (int ps = 0; ps < PASSES; ++ps)
        gv[ps] = ld_global_if(gate0 + gate_at[ps] + c, out_at[ps] != ~0u);
    };
    if (gate0) load_gates(0);
    // The maximum in use at the end, from the group of the last tile. The other group may still be reading this group's sums of the item before;
    // with two tiles or more it has published a maximum of this item since, and that was waited for. The owner of an item's only tile has
    // the maximum itself and waits for the item before in its place.
    const bool only = n_tiles == 1 && h == last && live > 0;
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(only ? bar_o_free : bar_m + 8 * last, (uint32_t)(only ? live - 1 : last_j >> 1) & 1, abort_flag));
    float end_m = -INFINITY;
    if (ok) {
      end_m = m_used[last * 128 + r];
      // a group that has seen no score: m = -inf and l = 0, or NaN where all of its scores were, which the sum has to show
      l_part[h * 128 + r] = m == -INFINITY ? l : l * ex2(m - end_m);
      mbar_arrive(bar_l);
      ok = __all_sync(0xffffffffu, mbar_wait(bar_l, (uint32_t)live & 1, abort_flag));
    }
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar_done, (uint32_t)live & 1, abort_flag));
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(full + 8 * e_slot, e_phase, abort_flag));
    if (ok) {
      tc_fence_after();
      const float sum = l_part[r] + l_part[128 + r];
      if (p.parts > 1 && h == 0) p.ws_ml[block_lin * 128 + r] = make_float2(end_m, sum);
      const float inv = p.parts > 1 ? 1.0f : sum == 0.f ? 0.f : 1.0f / sum;
      uint8_t* stage = smem + D::Q_BYTES + e_slot * SLOT + warp * (SLOT / 8);
      auto swz = [](int row) { return CH == 32 ? row & 7 : (row >> 1) & 3; };  // 16-byte chunks of a row: no two lanes of a quarter in one bank
#pragma unroll 1
      for (int c = 0; c < HD / 2; c += CH) {
        uint32_t v[CH];
        if constexpr (CH == 32) tmem_ld32(tmem + lanes + h * (HD / 2) + c, v);
        else tmem_ld16(tmem + lanes + h * (HD / 2) + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < LPR; ++i)
          *reinterpret_cast<float4*>(stage + lane * (CH * 4) + ((i ^ swz(lane)) * 16)) =
              make_float4(__uint_as_float(v[4 * i]) * inv, __uint_as_float(v[4 * i + 1]) * inv, __uint_as_float(v[4 * i + 2]) * inv, __uint_as_float(v[4 * i + 3]) * inv);
        __syncwarp();
        float4 o[PASSES];
#pragma unroll
        for (int ps = 0; ps < PASSES; ++ps) {
          const int row = ps * RPP + my_row;
          o[ps] = *reinterpret_cast<const float4*>(stage + row * (CH * 4) + ((my_c ^ swz(row)) * 16));
        }
        if (p.parts > 1) {
#pragma unroll
          for (int ps = 0; ps < PASSES; ++ps)
            if (out_at[ps] != ~0u)
              *reinterpret_cast<float4*>(p.ws_o + (block_lin * 128 + (warp & 3) * 32 + ps * RPP + my_row) * HD + h * (HD / 2) + c + my_c * 4) = o[ps];
        } else {
          if (gate0) {
#pragma unroll
            for (int ps = 0; ps < PASSES; ++ps) {
              const __nv_bfloat162* g2 = reinterpret_cast<const __nv_bfloat162*>(&gv[ps]);
              o[ps].x *= gate_of(__low2float(g2[0]));
              o[ps].y *= gate_of(__high2float(g2[0]));
              o[ps].z *= gate_of(__low2float(g2[1]));
              o[ps].w *= gate_of(__high2float(g2[1]));
            }
            if (c + CH < HD / 2) load_gates(c + CH);
          }
#pragma unroll
          for (int ps = 0; ps < PASSES; ++ps)
            st_global_if(out0 + out_at[ps] + c, make_uint2(pack_bf16(o[ps].x, o[ps].y), pack_bf16(o[ps].z, o[ps].w)), out_at[ps] != ~0u);
        }
        __syncwarp();
      }
      tc_fence_before();
      mbar_arrive(bar_o_free);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the slot goes back to TMA
      mbar_arrive(bar_e);
    }
    jj += n_tiles;
    ++live;
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
  constexpr int PER = HD / 32, U = 8;
  __shared__ int sums[4], found[3];
  if (threadIdx.x == 0) found[0] = -1;
  __syncthreads();
  const int all = scan_tiles(p, sums, [&](int b, int before, int n) {
    const int ti = blockIdx.x;
    if (ti < before || ti >= before + n) return;
    int off, len;
    tiles_of(p, b, off, len);
    found[0] = off;
    found[1] = (ti - before) * p.tokens;
    found[2] = min(p.tokens, len - found[1]);
  });
  __syncthreads();
  const int lane = threadIdx.x & 31, r = blockIdx.z * 4 + (threadIdx.x >> 5), G = p.G;
  if (all == 0 || found[0] < 0 || r >= found[2] * G) return;
  const int hg = blockIdx.y, kh = hg / p.sub, tt = r / G;
  const int head = kh * (p.heads / p.kv) + (hg - kh * p.sub) * G + r - tt * G;
  const size_t step = (size_t)gridDim.y * gridDim.x * 128, row0 = ((size_t)hg * gridDim.x + blockIdx.x) * 128 + r;
  float M = -INFINITY;
  float2 ml[4];  // parts lane, lane + 32, ... of at most 128
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int z = lane + 32 * k;
    ml[k] = z < parts ? p.ws_ml[z * step + row0] : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, ml[k].x);
  }
  M = warp_max(M);
  float acc[PER], sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (32 * k >= parts) break;
    // a part without keys, or one that this row sees nothing of, may have written no O: its sum is 0, and its row is not read. A sum of
    // NaN is none of these: it and its row count, at a weight of 0 too, so that a question whose keys are split shows a NaN as any other
    const bool some = ml[k].y != 0.f;
    const float wt = some ? ex2(ml[k].x - M) : 0.f;
    sum += wt * ml[k].y;
    const uint32_t have = __ballot_sync(0xffffffffu, some);
    const float* src = p.ws_o + (32 * k * step + row0) * HD + lane * PER;
    for (int z0 = 0; z0 < 32 && 32 * k + z0 < parts; z0 += U) {  // U rows are asked for before the first is used
      float2 v[U][PER / 2];
#pragma unroll
      for (int z = 0; z < U; ++z)
#pragma unroll
        for (int i = 0; i < PER / 2; ++i)
          v[z][i] = have >> (z0 + z) & 1u ? *reinterpret_cast<const float2*>(src + (size_t)(z0 + z) * step * HD + 2 * i) : make_float2(0.f, 0.f);
#pragma unroll
      for (int z = 0; z < U; ++z) {
        const float wz = __shfl_sync(0xffffffffu, wt, z0 + z);
#pragma unroll
        for (int i = 0; i < PER / 2; ++i) {
          acc[2 * i] += wz * v[z][i].x;
          acc[2 * i + 1] += wz * v[z][i].y;
        }
      }
    }
  }
  sum = warp_sum(sum);
  const size_t t = (size_t)found[0] + found[1] + tt;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const bf16* gate = p.gate_qg ? p.gate_qg + t * p.qg_stride + (size_t)(2 * head + 1) * HD + lane * PER : nullptr;
  bf16* dst = p.out + (t * p.heads + head) * HD + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; i += 2) {
    float a = acc[i] * inv, b = acc[i + 1] * inv;
    if (gate) {
      const __nv_bfloat162 g2 = *reinterpret_cast<const __nv_bfloat162*>(gate + i);
      a *= gate_of(__low2float(g2));
      b *= gate_of(__high2float(g2));
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
  int G, sub, tokens, parts;
  long long tiles;
  size_t state_bytes, ml_bytes, o_bytes;
};
Plan plan_of(int B, int T, int n_state, int heads, int kv, int hd) {
  Plan p;
  const int group = heads / kv;
  p.G = group;
  while (p.G > 128 || group % p.G != 0) --p.G;  // the rows of one token fit a tile
  p.sub = group / p.G;
  p.tokens = 128 / p.G;
  p.tiles = (long long)(T + p.tokens - 1LL) / p.tokens + B;
  // split the keys where there is no CTA for every SM and the state is at least eight tiles long: about two CTAs per SM, at least
  // two key tiles per part
  const long long ctas = p.tiles * kv * p.sub;
  const int st_tiles = (int)((n_state + KT - 1LL) / KT), sms = sm_count();
  p.parts = 1;
  if (ctas <= sms && st_tiles >= 8) p.parts = max(1, min(min(2 * sms / (int)ctas, st_tiles / 2), 128));
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
  p.parts = pl.parts;
  p.max_tiles = (int)pl.tiles;
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
  // one CTA per SM, more only where one would have more items than its table holds
  const long long items = pl.tiles * a.kv * pl.sub * pl.parts;
  if (items > (1 << 30)) return cudaErrorInvalidValue;
  const unsigned grid = (unsigned)max(min(items, (long long)sm_count()), (items + MAX_ITEMS - 1) / MAX_ITEMS);
  auto map = [](const TcTensorMap& m) -> const CUtensorMap& { return *reinterpret_cast<const CUtensorMap*>(&m); };
  // started while the state is still being decoded: the setup of barriers and TMEM and the search for the items lie under that, every load waits
  // for it (one question of 16 tokens over 4096 rows: 25.9 -> 24.0 us; with the merge started like this as well 29.3, and the same for
  // the new tokens' merge gained nothing)
  if (a.n_state > 0) CUDA_TRY(launch_dependent(kv4_attention_kernel<HD>, grid, NUM_THREADS, Shape<HD>::SMEM, s, map(q), map(ksm), map(vsm), map(ko), map(vo), p));
  else kv4_attention_kernel<HD><<<grid, NUM_THREADS, Shape<HD>::SMEM, s>>>(map(q), map(ksm), map(vsm), map(ko), map(vo), p);
  CUDA_TRY(cudaGetLastError());
  if (pl.parts > 1) kv4_attention_merge_kernel<HD><<<dim3((unsigned)pl.tiles, a.kv * pl.sub, 32), 128, 0, s>>>(p, pl.parts);
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
