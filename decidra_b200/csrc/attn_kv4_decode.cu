// Attention of the newest tokens of many sequences over their stretches of a 4-bit K/V cache (dcd_k_attention_kv4_decode).
//
// A pair is a sequence with up to four neighbouring K/V heads (and, for more query rows than a warp holds, one round of them); its keys
// come in blocks of 32. All blocks of all pairs lie behind each other and every CTA of one resident wave takes the same number of
// them, so sequences of very different lengths keep every SM busy to the end, and a CTA pays its start (offsets, Q, the first loads)
// once or twice instead of once per chunk of keys. A warp has one of the heads (with fewer than four, the warps of a head take its
// blocks in turn), so that a CTA reads whole rows of the cache: one head's 128 bytes of every 512, and 16 of every 64 bytes of scales,
// cost 17 % more DRAM traffic than they hold. Each warp has room for one block of its own in shared memory (cp.async, no barrier between
// warps): the next K is on its way from the end of the S products on, the next V from the end of the P.V products, so that half a block
// per warp is always in flight and twelve warps fit on an SM (two and three whole blocks a warp and eight warps: 162 us where this takes
// 144, half of the issue slots empty). Few query rows share each key (tokens x heads of the group, eight per MMA column tile), so the
// kernel lives on getting 0.5625 bytes a value from HBM into matrix fragments:
//   S^T[16 keys, 8 rows]  += K[16 keys, 16 dims] Q^T      mma.m16n8k16 with the KEYS as the 16-row operand: all of it is used
//   O^T[16 dims, 8 rows]  += V^T[16 dims, 16 keys] P^T    even for one token of six heads, where rows as M would fill 6 of 16
// The fragments are made in registers straight from the code words. The order of the contracted dimensions is free as long as Q has
// the same, so a lane's K values are 16 (head_dim 64) to 64 (256) consecutive dimensions of two keys, loaded 16 bytes at a time; a
// lane's V values are 8 to 32 consecutive dimensions of four keys, and the code words of two neighbouring keys are merged nibble by
// nibble first, so that one conversion instruction (cvt.rn.f16x2.e2m1x2, which picks its byte for free: 182 values per ns and SM
// measured with the scale's product, against 63 for shifting bits into place and 79 needed at HBM speed) gives the pair (key, key + 1)
// of one dimension that the fragment wants. code * scale is exact in f16. P^T comes from S^T with one 8 x 8 transpose per 16 keys.
//
// Q is bf16 and the products f16: each row is divided by the power of two of its largest value (exact but for elements below 2^-14 of
// it, which keep an absolute error of 2^-25 of it), and the factor returns in the softmax scale. P is held as p * 2^10 in f16, so
// that weights down to 2^-34 of the row's largest survive. Maxima, sums and O are f32.
//
// What bounds it: 64 sequences of 1024 to 16384 rows of 4 heads of 256 take 144 to 170 us, one machine and another, 4.4 to 3.7 TB/s (97 us at
// the copy rate). Of 1190 instructions per 32 keys and head 512 convert and scale codes; 0.57 are issued a cycle and scheduler, the ALU
// pipe is 54 % busy, and 5 % of the stalls wait for memory: the registers hold three warps a scheduler, and no more of them would fit.
// One token over 2048 rows takes 12.2 to 15 us, all latency.
//
// Rows whose keys all went through one warp are finished there; otherwise each warp leaves its unnormalised O with maximum and sum in the
// workspace, and a second kernel adds them up in their order. Keys beyond the stretch are zero-filled, masked keys get p = 0; a sum of 0 is a
// token that sees no row, a sum of NaN stays NaN.
#include "common.cuh"
#include "kv4.h"

namespace kvd {

constexpr int KB = 32;
constexpr float P_SHIFT = 10.0f;  // P is held as p * 2^10

constexpr int WARPS = 4;
// CTAs per SM, Q fragments in shared memory where registers run out
constexpr int ctas_of(int nt) { return nt == 1 ? 3 : 2; }
template <int HD, int NT> struct Cfg {
  static constexpr int CTAS = ctas_of(NT);
  static constexpr bool Q_SMEM = NT * HD >= 256;
};

template <int HD> struct Block {
  static constexpr int ROW = HD / 2, SROW = HD / 16;                            // bytes of a key's codes and scales
  static constexpr int K = 0, V = KB * ROW, KS = 2 * KB * ROW, VS = KS + KB * SROW;
  static constexpr int BYTES = VS + KB * SROW;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool valid) {  // zeros where !valid
  const int n = valid ? N : 0;
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// the four byte pairs of codes in w as f16x2 (low nibble in the low half)
__device__ __forceinline__ void e2m1x8(uint32_t w, uint32_t (&v)[4]) {
  asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b1;\ncvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
      : "r"(w));
}
__device__ __forceinline__ uint32_t e4m3x2(uint32_t two) {  // two scales (low 16 bits) as f16x2
  uint32_t r;
  asm("{\n.reg .b16 h, t;\nmov.b32 {h, t}, %1;\ncvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t hmul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) { return __byte_perm(a, b, s); }

// Shared-memory position of 16-byte chunk `c` of key `k`: a quarter-warp reads two keys' four chunks (K) or four keys' two (V), which
// for rows of 128 bytes would meet in the same banks.
template <int HD> __device__ __forceinline__ int k_chunk(int k, int c) { return HD == 256 ? c ^ ((k & 1) << 2) : c; }
template <int HD> __device__ __forceinline__ int v_chunk(int k, int c) { return HD == 256 ? c ^ (k & 6) : HD == 128 ? c ^ (k & 2) : c; }

struct Args {
  Kv4DecodeArgs a;
  int hc;          // K/V heads of a pair: 4, 2 or 1
  int q_min;       // least blocks per CTA
  uint32_t split;  // places of pairs that are split between CTAs; the others' are behind them
  float* ws_o;     // [places][hd] unnormalised O of a part of a row
  float2* ws_ml;   // [places] (maximum in log2 units, sum)
  uint2* ws_n;     // [T * heads] the row's parts and the place of its first: they lie behind each other
  int* ws_falls;   // some sequence's offsets fall or leave the batch
};

// The first place of a row of a pair that is split between CTAs from `first_cta` on. A warp's row has a place for every even number of a CTA
// and every odd one: the parts of a pair go to 2 first_cta and the numbers behind it, and the next pair that is split begins in the last CTA
// of this one or later, so that twice its number is above all of them. That bounds the places by the CTAs, whatever the lengths are and however many
// parts a row has.
__device__ __forceinline__ uint32_t split_place(int row, int first_cta, int step) { return ((uint32_t)row * gridDim.x + first_cta) * (2 * step); }

struct Sequence {
  bool sound;  // its offsets
  int off, L, len;
  size_t start;
};
// Bounds-checked view of sequence b; a bad one has no tokens or no rows.
__device__ __forceinline__ Sequence sequence(const Kv4DecodeArgs& a, int b, bool report) {
  Sequence s;
  s.off = a.cu[b];
  const int stop = a.cu[b + 1];
  s.sound = s.off >= 0 && stop >= s.off && stop <= a.T;  // compared before they are subtracted: the difference of bad ones may overflow
  s.L = s.sound ? stop - s.off : 0;
  if (!s.sound && report) set_err(a.err, DERR_OFFSETS);
  const int64_t st = a.seg_start[b];
  s.len = a.seg_len[b];
  s.start = (size_t)st;
  if (st < 0 || s.len < 0 || s.len > a.max_len || (uint64_t)st > a.cache_rows || (uint64_t)s.len > a.cache_rows - (uint64_t)st) {
    if (report) set_err(a.err, DERR_CACHE_ROW);
    s.len = 0;
    s.start = 0;
  }
  return s;
}

// Block numbers are 64-bit; what is divided in earnest fits 32, where a division is a tenth of the 64-bit one.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return (((unsigned long long)a | (unsigned long long)b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

template <int ROWS>
__device__ __forceinline__ int rounds_of(const Sequence& s, int G) { return (s.L * G + ROWS - 1) / ROWS; }
// Blocks of one pair of the sequence: at least one, so that the tokens of an empty stretch get their zeros.
__device__ __forceinline__ int blocks_of(const Sequence& s) { return max(1, (s.len + KB - 1) / KB); }

// PER consecutive values of a row from dimension d: normalised, gated, rounded once; stored N at a time
template <int PER>
__device__ __forceinline__ void store_row(const Kv4DecodeArgs& a, const float (&acc)[PER], float sum, size_t at, int t, int h, int hd, int d) {
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // 0: a token that sees no row; NaN stays
  const bf16* gate = a.gate_qg ? a.gate_qg + (size_t)t * a.qg_stride + (size_t)(2 * h + 1) * hd + d : nullptr;
  bf16* out = a.out + at * hd + d;
  constexpr int N = PER < 8 ? PER : 8;
  struct alignas(2 * N) Values {
    __nv_bfloat162 two[N / 2];
  };
#pragma unroll
  for (int i = 0; i < PER; i += N) {
    Values gv, v;
    if (gate) gv = *reinterpret_cast<const Values*>(gate + i);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      float x = acc[i + j] * inv, y = acc[i + j + 1] * inv;
      if (gate) {
        x *= sigmoid_f(__low2float(gv.two[j / 2]));
        y *= sigmoid_f(__high2float(gv.two[j / 2]));
      }
      v.two[j / 2] = __floats2bfloat162_rn(x, y);
    }
    *reinterpret_cast<Values*>(out + i) = v;
  }
}

template <int HD, int NT>
__global__ void __launch_bounds__(WARPS * 32, Cfg<HD, NT>::CTAS) kv4_decode_kernel(const Args p) {
  using R = Block<HD>;
  constexpr int KW = HD / 32;               // K code words of a lane per key
  constexpr int KL = KW < 4 ? KW : 4;       // ... loaded at once
  constexpr int VW = HD / 64;               // V code words of a lane per key
  constexpr int ROWS = 8 * NT;
  constexpr bool Q_SMEM = Cfg<HD, NT>::Q_SMEM;
  const Kv4DecodeArgs& a = p.a;
  const int G = a.heads / a.kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int hc = p.hc, n_groups = a.kv / hc, my_head = warp % hc, first = warp / hc, step = WARPS / hc;  // this warp's head of a pair, and its blocks
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* const st = smem + warp * R::BYTES;
  const uint32_t st_addr = smem_addr(st);
  uint2* q_smem = reinterpret_cast<uint2*>(smem + WARPS * R::BYTES) + warp * (HD / 16 * NT * 32);  // [word * 2 + half][nt][lane]
  const float scale_log2e = (1.0f / sqrtf((float)HD)) * 1.4426950408889634f;

  // ---- this CTA's blocks: thread t adds up the sequences [t * per, (t + 1) * per), then a scan over the threads ------------------------------
  __shared__ long long sums[WARPS];
  __shared__ int at_b;
  __shared__ long long at_u;
  long long u, u_end, quota;
  int b;
  {
    const int per = (a.B + WARPS * 32 - 1) / (WARPS * 32), b0 = min((int)threadIdx.x * per, a.B), b1 = min(b0 + per, a.B);
    long long mine = 0;
    int falls = 0;
    for (int i = b0; i < b1; ++i) {
      const Sequence s = sequence(a, i, blockIdx.x == 0);
      falls |= !s.sound;
      mine += (long long)n_groups * rounds_of<ROWS>(s, G) * blocks_of(s);
    }
    if (blockIdx.x == 0) {
      falls = __syncthreads_or(falls);
      if (threadIdx.x == 0) *p.ws_falls = falls;
    }
    long long before = mine, total = 0;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, before, i);
      if (lane >= i) before += x;
    }
    if (lane == 31) sums[warp] = before;
    before -= mine;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i < warp) before += sums[i];
      total += sums[i];
    }
    quota = max(quotient(total + gridDim.x - 1, gridDim.x), (long long)p.q_min);
    u = quota * blockIdx.x;
    u_end = min(total, u + quota);
    if (u >= u_end) return;
    if (before <= u && u < before + mine) {  // one thread: its range holds the first block
      int i = b0;
      for (; i < b1; ++i) {
        const Sequence s = sequence(a, i, false);
        const long long n = (long long)n_groups * rounds_of<ROWS>(s, G) * blocks_of(s);
        if (u < before + n) break;
        before += n;
      }
      at_b = i;
      at_u = before;
    }
    __syncthreads();
    b = at_b;
  }
  long long seq_u = at_u;  // first block of sequence b
  Sequence sq = sequence(a, b, false);

  while (u < u_end) {
    const int nblk = blocks_of(sq), n_rows = sq.L * G;
    const long long in_seq = u - seq_u;
    if (in_seq >= (long long)n_groups * rounds_of<ROWS>(sq, G) * nblk) {
      seq_u += (long long)n_groups * rounds_of<ROWS>(sq, G) * nblk;
      sq = sequence(a, ++b, false);
      continue;
    }
    const int pair = (int)quotient(in_seq, nblk), kh = pair % n_groups * hc + my_head, r0 = pair / n_groups * ROWS, first_blk = (int)(in_seq - (long long)pair * nblk);
    const int n_blocks = (int)min((long long)(nblk - first_blk), u_end - u);
    const long long pair_u = u - first_blk;
    const int first_cta = (int)quotient(pair_u, quota), n_parts = (int)quotient(pair_u + nblk - 1, quota) - first_cta + 1, part = (int)blockIdx.x - first_cta;
    u += n_blocks;
    const int k0 = first_blk * KB, k1 = min(sq.len, k0 + n_blocks * KB);  // the keys of this part, relative to the stretch

    // rows of the cache for this head
    const size_t row0 = (sq.start + (size_t)k0) * a.kv + kh;
    const uint8_t* kc = a.cache.k.codes + row0 * R::ROW;
    const uint8_t* vc = a.cache.v.codes + row0 * R::ROW;
    const uint8_t* ks = a.cache.k.scales + row0 * R::SROW;
    const uint8_t* vs = a.cache.v.scales + row0 * R::SROW;
    const size_t code_step = (size_t)a.kv * R::ROW, scale_step = (size_t)a.kv * R::SROW;

    // K or V of a block: lane (key, chunk) takes every KPL-th key's 16 bytes; addresses advance by additions
    constexpr int CHUNKS = R::ROW / 16, KPL = 32 / CHUNKS;
    const int f_key = lane / CHUNKS, f_chunk = lane % CHUNKS;
    const size_t lane_code = f_key * code_step + f_chunk * 16, lane_scale = lane * scale_step, pass_step = KPL * code_step;
    auto fetch = [&](int blk, bool second) {
      const int left = (k1 - k0) - blk * KB;  // keys of the block that exist
      const uint8_t* codes = (second ? vc : kc) + (size_t)blk * KB * code_step;
      const uint8_t* scales = (second ? vs : ks) + (size_t)blk * KB * scale_step;
      const uint32_t to = st_addr + (second ? R::V : R::K), to_scales = st_addr + (second ? R::VS : R::KS) + lane * R::SROW;
      const uint8_t* from = codes + lane_code;
      if (left >= KB) {
#pragma unroll
        for (int i = 0; i < KB / KPL; ++i) {
          const int key = i * KPL + f_key;
          cp_async<16>(to + key * R::ROW + (second ? v_chunk<HD>(key, f_chunk) : k_chunk<HD>(key, f_chunk)) * 16, from, true);
          from += pass_step;
        }
        cp_async<R::SROW>(to_scales, scales + lane_scale, true);
      } else {  // zeros behind the last key
#pragma unroll 1
        for (int i = 0; i < KB / KPL; ++i) {
          const int key = i * KPL + f_key;
          cp_async<16>(to + key * R::ROW + (second ? v_chunk<HD>(key, f_chunk) : k_chunk<HD>(key, f_chunk)) * 16, key < left ? from : codes, key < left);
          from += pass_step;
        }
        cp_async<R::SROW>(to_scales, lane < left ? scales + lane_scale : scales, lane < left);
      }
    };

    // ---- Q is asked for in front of the first block: behind all CTAs' first blocks it would come last -----------------------------
    uint4 qw[NT][KW];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = r0 + nt * 8 + g;
      const bool live = row < n_rows;
      const bf16* src = live ? a.q + (size_t)(sq.off + row / G) * a.q_stride + (size_t)(kh * G + row % G) * HD : a.q;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const int d = HD == 256 ? (w >> 2) * 128 + 32 * c + 8 * (w & 3) : KL * 8 * c + 8 * w;
        qw[nt][w] = live ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
      }
    }
    if (first < n_blocks) fetch(first, false);
    cp_commit();
    if (first < n_blocks) fetch(first, true);
    cp_commit();
    // ---- Q as the column operand: lane (g, c) holds row g's dimensions of quad position c -------------
    uint2 qf[Q_SMEM ? 1 : NT][Q_SMEM ? 1 : KW * 2];
    float f[NT][2];  // softmax factor of rows 2c, 2c + 1
    int end[NT][2];  // first key (relative to the chunk) that the row does not see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float m = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&qw[nt][w]);
#pragma unroll
        for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fabsf(__low2float(h[i])), fabsf(__high2float(h[i]))));
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // 2^e <= m < 2^(e+1); a row of zeros and one of infinities keep their values
      const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -126), 126);
      const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&qw[nt][w]);
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = pack_f16(__low2float(h[i]) * inv, __high2float(h[i]) * inv);
        if constexpr (Q_SMEM) {
          q_smem[((2 * w) * NT + nt) * 32 + lane] = make_uint2(v[0], v[1]);
          q_smem[((2 * w + 1) * NT + nt) * 32 + lane] = make_uint2(v[2], v[3]);
        } else {
          qf[nt][2 * w] = make_uint2(v[0], v[1]);
          qf[nt][2 * w + 1] = make_uint2(v[2], v[3]);
        }
      }
      const float fr = scale_log2e * __uint_as_float((uint32_t)(127 + e) << 23);
      f[nt][0] = __shfl_sync(0xffffffffu, fr, 8 * c);
      f[nt][1] = __shfl_sync(0xffffffffu, fr, 8 * c + 4);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rr = min(r0 + nt * 8 + 2 * c + i, n_rows - 1);
        end[nt][i] = min(sq.len - (sq.L - 1 - rr / G), k1) - k0;
      }
    }
    if constexpr (Q_SMEM) __syncwarp();

    float o[HD / 16][NT][4];
#pragma unroll
    for (int t = 0; t < HD / 16; ++t)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][nt][i] = 0.f;
    float m[NT][2], l[NT][2];
    int first_end = end[0][0];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[nt][i] = -INFINITY;
        l[nt][i] = 0.f;
        first_end = min(first_end, end[nt][i]);
      }

    for (int blk = first; blk < n_blocks; blk += step) {
      cp_wait<1>();  // K; V may still be under way
      __syncwarp();
      // ---- S^T of two 16-key tiles ------------------------------------------------------------------
      float s[2][NT][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][nt][i] = 0.f;
#pragma unroll
      for (int ld = 0; ld < KW / KL; ++ld) {
        uint32_t w[4][KL];   // [tile * 2 + (key + 8)][word]
        uint32_t sc[4];      // the keys' scales of this load, f16x2
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = (i >> 1) * 16 + (i & 1) * 8 + g;
          if constexpr (KL == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(st + R::K + key * R::ROW + k_chunk<HD>(key, ld * 4 + c) * 16);
            w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
            sc[i] = e4m3x2(*reinterpret_cast<const uint16_t*>(st + R::KS + key * R::SROW + ld * 8 + 2 * c));
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(st + R::K + key * R::ROW + c * 8);
            w[i][0] = u.x; w[i][1] = u.y;
            sc[i] = e4m3x2((uint32_t)st[R::KS + key * R::SROW + c]);
          }
        }
#pragma unroll
        for (int wi = 0; wi < KL; ++wi) {
          uint32_t av[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t s2 = prmt(sc[i], 0, wi < 2 ? 0x1010 : 0x3232);  // two words share a scale
            e2m1x8(w[i][wi], av[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) av[i][j] = hmul(av[i][j], s2);
          }
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int step = (ld * KL + wi) * 2 + half;
              const uint2 q = Q_SMEM ? q_smem[(step * NT + nt) * 32 + lane] : qf[Q_SMEM ? 0 : nt][Q_SMEM ? 0 : step];
#pragma unroll
              for (int t = 0; t < 2; ++t) mma(s[t][nt], av[2 * t][2 * half], av[2 * t + 1][2 * half], av[2 * t][2 * half + 1], av[2 * t + 1][2 * half + 1], q.x, q.y);
            }
        }
      }

      __syncwarp();
      if (blk + step < n_blocks) fetch(blk + step, false);
      cp_commit();

      // ---- softmax: lane (g, c) has keys g, g + 8 of either tile for rows 2c, 2c + 1 --------------------
      const int j0 = blk * KB;
      const bool partial = j0 + KB > first_end;
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = s[t][nt][i] * f[nt][i & 1];
            if (partial && j0 + t * 16 + (i >> 1) * 8 + g >= end[nt][i & 1]) x = -INFINITY;
            s[t][nt][i] = x;
            mx[i & 1] = fmaxf(mx[i & 1], x);
          }
        float corr[2], neg[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 4));
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 8));
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 16));
          mx[i] = fmaxf(mx[i], m[nt][i]);
          const float base = mx[i] == -INFINITY ? 0.f : mx[i];  // a row that has seen nothing yet
          corr[i] = ex2(m[nt][i] - base);
          neg[i] = P_SHIFT - base;
          l[nt][i] *= corr[i];
        }
        if (__any_sync(0xffffffffu, mx[0] != m[nt][0] || mx[1] != m[nt][1])) {
#pragma unroll
          for (int t = 0; t < HD / 16; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][nt][i] *= corr[i & 1];
        }
        m[nt][0] = mx[0];
        m[nt][1] = mx[1];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[i] = ex2(s[t][nt][i] + neg[i & 1]);
            l[nt][i & 1] += e[i];
          }
          pb[t][nt][0] = transpose8(pack_f16(e[0], e[1]));
          pb[t][nt][1] = transpose8(pack_f16(e[2], e[3]));
        }
      }

      cp_wait<1>();  // V; the next K may still be under way
      __syncwarp();
      // ---- O^T += V^T P^T: lane (g, c) holds 8 to 32 dimensions of keys 2c, 2c + 1, 2c + 8, 2c + 9 ---------
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        uint32_t pt[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          pt[nt][0] = t ? pb[1][nt][0] : pb[0][nt][0];
          pt[nt][1] = t ? pb[1][nt][1] : pb[0][nt][1];
        }
        uint32_t w[4][VW], sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = t * 16 + 2 * c + (i & 1) + (i >> 1) * 8;
          if constexpr (HD == 256) {
            const uint4 u = *reinterpret_cast<const uint4*>(st + R::V + key * R::ROW + v_chunk<HD>(key, g) * 16);
            w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
            sc[i] = *reinterpret_cast<const uint16_t*>(st + R::VS + key * R::SROW + 2 * g);
          } else if constexpr (HD == 128) {
            const uint2 u = *reinterpret_cast<const uint2*>(st + R::V + key * R::ROW + v_chunk<HD>(key, g >> 1) * 16 + (g & 1) * 8);
            w[i][0] = u.x; w[i][1] = u.y;
            sc[i] = st[R::VS + key * R::SROW + g];
          } else {
            w[i][0] = *reinterpret_cast<const uint32_t*>(st + R::V + key * R::ROW + g * 4);
            sc[i] = st[R::VS + key * R::SROW + (g >> 1)];
          }
        }
        uint32_t s01[2], s89[2];  // per scale group of the lane: (key, key + 1)
        if constexpr (HD == 256) {
          const uint32_t x0 = e4m3x2(sc[0]), x1 = e4m3x2(sc[1]), x2 = e4m3x2(sc[2]), x3 = e4m3x2(sc[3]);
          s01[0] = prmt(x0, x1, 0x5410); s01[1] = prmt(x0, x1, 0x7632);
          s89[0] = prmt(x2, x3, 0x5410); s89[1] = prmt(x2, x3, 0x7632);
        } else {
          s01[0] = s01[1] = e4m3x2(sc[0] | sc[1] << 8);
          s89[0] = s89[1] = e4m3x2(sc[2] | sc[3] << 8);
        }
#pragma unroll
        for (int wi = 0; wi < VW; ++wi) {
          // the two keys' codes of one dimension side by side in a byte: even dimensions, odd dimensions
          constexpr uint32_t LO = 0x0F0F0F0Fu, HI = 0xF0F0F0F0u;
          uint32_t ev[4], ov[4], ev8[4], ov8[4];
          e2m1x8((w[0][wi] & LO) | ((w[1][wi] << 4) & HI), ev);
          e2m1x8(((w[0][wi] >> 4) & LO) | (w[1][wi] & HI), ov);
          e2m1x8((w[2][wi] & LO) | ((w[3][wi] << 4) & HI), ev8);
          e2m1x8(((w[2][wi] >> 4) & LO) | (w[3][wi] & HI), ov8);
          const uint32_t sa = s01[HD == 256 ? wi >> 1 : 0], sb = s89[HD == 256 ? wi >> 1 : 0];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a0 = hmul(ev[j], sa), a1 = hmul(ov[j], sa), a2 = hmul(ev8[j], sb), a3 = hmul(ov8[j], sb);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma(o[wi * 4 + j][nt], a0, a1, a2, a3, pt[nt][0], pt[nt][1]);
          }
        }
      }
      __syncwarp();
      if (blk + step < n_blocks) fetch(blk + step, true);
      cp_commit();
    }
    cp_wait<0>();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], 4);
        l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], 8);
        l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], 16);
      }
    // ---- every warp is a part of its rows and writes it from registers: lane (g, c) holds the HD / 8 dimensions from g * (HD / 8) on,
    // two per t, of rows 2c, 2c + 1. (With a head's warps added up through shared memory first, 64 sequences took 147 us instead of 144,
    // and nine of four drafted tokens over two heads the same 33: the second kernel has fewer parts then, this one three barriers.)
    const int parts_all = n_parts * step, my_part = part * step + first;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = r0 + nt * 8 + 2 * c + i;
        if (r >= n_rows) continue;
        const int tt = r / G, tok = sq.off + tt, h = kh * G + r - tt * G;
        const size_t at = (size_t)tok * a.heads + h;
        const uint32_t base = n_parts == 1 ? p.split + (uint32_t)at * step : split_place(my_head * ROWS + r - r0, first_cta, step);
        if (my_part == 0 && g == 0) p.ws_n[at] = make_uint2(parts_all, base);
        if (parts_all > 1) {
          if (g == 0) p.ws_ml[base + my_part] = make_float2(m[nt][i], l[nt][i]);
          float* dst = p.ws_o + (size_t)(base + my_part) * HD + g * (HD / 8);
#pragma unroll
          for (int t = 0; t < HD / 16; t += 2)
            *reinterpret_cast<float4*>(dst + 2 * t) = make_float4(o[t][nt][i], o[t][nt][i + 2], o[t + 1][nt][i], o[t + 1][nt][i + 2]);
        } else {
          float acc[HD / 8];
#pragma unroll
          for (int t = 0; t < HD / 16; ++t) {
            acc[2 * t] = o[t][nt][i];
            acc[2 * t + 1] = o[t][nt][i + 2];
          }
          store_row<HD / 8>(a, acc, l[nt][i], at, tok, h, HD, g * (HD / 8));
        }
      }
    __syncwarp();  // before the next pair's Q and blocks come
  }
}

// out = sum_z O_z 2^(m_z - M) / sum_z l_z 2^(m_z - M). W warps per (token, head) take the parts in turn; their sums are added in
// order. The row's sequence is found 32 offsets at a time, 32 parts' weights come at once, and the rows of four or eight parts are asked
// for before the first is used: a chain of loads is what this kernel's time is made of (both kernels, one token over 8000 rows in 125
// parts: 14.7 us, over 2048 rows 12.4; when a row's parts lay further apart 17 and 12.7, and with a loop of one part after the other and never
// more than four warps 23.5 and 14.3).
template <int HD, int W>
__global__ void __launch_bounds__(W > 4 ? W * 32 : 128) kv4_decode_merge_kernel(const Args p) {
  constexpr int WARPS_HERE = W > 4 ? W : 4, VEC = HD == 64 ? 2 : 4, NV = HD / 32 / VEC, U = W > 4 ? 8 : 4;  // a lane's values: VEC from lane * VEC on, NV times
  struct alignas(4 * VEC) Values {
    float f[VEC];
  };
  __shared__ float part[W > 1 ? WARPS_HERE : 1][HD], part_sum[WARPS_HERE];
  const Kv4DecodeArgs& a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp % W;
  const size_t at = (size_t)blockIdx.x * (WARPS_HERE / W) + warp / W;
  const int t = (int)(at / (unsigned)a.heads), h = (int)(at - (size_t)t * a.heads);
  int nz = 0;
  size_t base = 0;
  if (t < a.T) {
    int lo = 0, hi = a.B;  // cu[lo] <= t, and t < cu[hi] where it is in a sequence at all
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, i = min(lo + (lane + 1) * step, hi);
      const unsigned below = __ballot_sync(0xffffffffu, i < hi && a.cu[i] <= t);
      const int n = __popc(below);  // offsets rise
      hi = min(lo + (n + 1) * step, hi);
      lo += n * step;
    }
    auto has = [&](int i) {  // sequence i is sound and t one of its tokens
      const int off = a.cu[i], end = a.cu[i + 1];
      return off >= 0 && off <= t && t < end && end <= a.T;
    };
    bool mine = has(lo);
    // not there: a row behind the last sequence, or, where some offsets fall, one of a sound sequence that was missed
    if (!mine && *p.ws_falls)
      for (int i = lane; !mine && i - lane < a.B; i += 32) mine = __any_sync(0xffffffffu, i < a.B && has(i));
    if (mine) {
      const uint2 n = p.ws_n[at];
      nz = (int)n.x;
      base = n.y;
    }
  }
  if (W == 1 && nz <= 1) return;  // finished by its only warp, or no token of a sequence
  const float2* ml = p.ws_ml + base;
  float M = -INFINITY;
#pragma unroll 4
  for (int z = lane; z < nz; z += 32) M = fmaxf(M, ml[z].x);
  M = warp_max(M);
  float acc[NV][VEC], sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[i][j] = 0.f;
  if (nz > 1) {
    const float* src = p.ws_o + base * HD + lane * VEC;
    for (int z0 = w; z0 < nz; z0 += 32 * W) {  // this warp's next 32 parts: z0, z0 + W, ...
      const int mine = z0 + lane * W;
      const float2 x = mine < nz ? ml[mine] : make_float2(-INFINITY, 0.f);
      // a part that saw nothing has m = -inf and sum 0: weight 0 on zeros. One whose scores are all NaN has m = -inf and sum NaN, which stays
      const float wt = x.y == 0.f ? 0.f : ex2(x.x - M);
      sum += wt * x.y;
      const int n = min(32, (nz - z0 + W - 1) / W);
      for (int z = 0; z < n; z += U) {
        Values v[U][NV];
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            if (z + k < n) {
              v[k][i] = *reinterpret_cast<const Values*>(src + (size_t)(z0 + (z + k) * W) * HD + i * 32 * VEC);
            } else {
#pragma unroll
              for (int j = 0; j < VEC; ++j) v[k][i].f[j] = 0.f;
            }
          }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const float wz = __shfl_sync(0xffffffffu, wt, (z + k) & 31);
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[i][j] += wz * v[k][i].f[j];
        }
      }
    }
    sum = warp_sum(sum);
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) part[warp][(i * 32 + lane) * VEC + j] = acc[i][j];
    if (lane == 0) part_sum[warp] = sum;
    __syncthreads();
    if (w != 0 || nz <= 1) return;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[i][j] = 0.f;
#pragma unroll
    for (int v = 0; v < W; ++v) {
      sum += part_sum[warp + v];
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[i][j] += part[warp + v][(i * 32 + lane) * VEC + j];
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) store_row<VEC>(a, acc[i], sum, at, t, h, HD, (i * 32 + lane) * VEC);
}

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return 148;
  return sms;
}

// How a call is cut up. The blocks per CTA follow the lengths on the device: max_len only bounds the CTAs and parts of a small call, so that
// a bound far above the lengths costs neither time nor memory. (With a least share that grew with B * max_len, 64 sequences of about 1000
// rows took 393 us under a bound of 131072, where they take 35 under any, and one of 100000 rows among 199 short ones 1215, now 89.)
struct Plan {
  int hc, nt, grid, q_min;  // K/V heads of a pair, column tiles of eight rows, CTAs, least blocks per CTA
  int parts;                // of a row, where the sequences are about as long as each other
  size_t split, places;     // places of parts: of the pairs split between CTAs, and all
};
Plan plan_of(int B, int T, int max_len, int heads, int kv, int hd) {
  Plan p;
  p.hc = kv % 4 == 0 ? 4 : kv % 2 == 0 ? 2 : 1;
  // column tiles by the rows of a sequence of average length; longer ones take several rounds over their keys
  const long long rows = ((long long)T + B - 1) / B * (heads / kv);
  p.nt = rows <= 8 ? 1 : rows <= 16 || hd == 256 ? 2 : 4;
  const int sms = sm_count(), wave = sms * ctas_of(p.nt), step = WARPS / p.hc;
  p.q_min = 2 * step;  // two per warp
  const long long pairs = (kv / p.hc) * ((long long)T * (heads / kv) / (8 * p.nt) + B), blocks = max(1LL, ((long long)max_len + KB - 1) / KB);
  p.grid = (double)pairs * (double)blocks >= (double)wave * p.q_min ? wave : (int)((pairs * blocks + p.q_min - 1) / p.q_min);
  p.parts = (int)min((blocks + p.q_min - 1) / p.q_min + 1, p.grid / pairs + 2) * step;
  // no more with more tokens, sequences or rows than the workspace of the largest call holds: sized for the column tiles that a call of the same
  // heads may take at most (grid * nt <= units)
  const int nt_max = hd == 256 ? 2 : 4;
  const double units = (kv / p.hc) * ((double)T * (heads / kv) / 8 + (double)B * nt_max) * (double)blocks / p.q_min + nt_max;
  p.split = (size_t)2 * WARPS * 8 * (size_t)min(ceil(units), (double)sms * ctas_of(nt_max) * nt_max);
  p.places = p.split + (step > 1 ? (size_t)T * heads * step : 0);
  return p;
}

template <int HD, int NT>
cudaError_t run(const Args& p, const Plan& plan, cudaStream_t s) {
  using C = Cfg<HD, NT>;
  constexpr int bytes = WARPS * (Block<HD>::BYTES + (C::Q_SMEM ? HD / 16 * NT * 256 : 0));
  static_assert(C::CTAS * (bytes + 1024 + 256) <= 228 * 1024, "shared memory of an SM");
  CUDA_TRY(cudaFuncSetAttribute(kv4_decode_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  kv4_decode_kernel<HD, NT><<<plan.grid, WARPS * 32, bytes, s>>>(p);
  CUDA_TRY(cudaGetLastError());
  const size_t rows = (size_t)p.a.T * p.a.heads;
  // More warps a row where more parts make a longer chain; fewer where they would have less than a part or two each (256 sequences of
  // about 1000 rows, most of them of one part: 83 us with a warp a row, 94 with four; one of 100000 among 199 short ones 89 and 69)
  if (plan.parts <= 8) kv4_decode_merge_kernel<HD, 1><<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(p);
  else if (plan.parts <= 32) kv4_decode_merge_kernel<HD, 4><<<(unsigned)rows, 128, 0, s>>>(p);
  else kv4_decode_merge_kernel<HD, 16><<<(unsigned)rows, 512, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace kvd

size_t kv4_decode_workspace(int B, int T, int max_len, int heads, int kv, int hd) {
  const kvd::Plan p = kvd::plan_of(B, T, max_len, heads, kv, hd);
  return p.places * ((size_t)hd * sizeof(float) + sizeof(float2)) + (size_t)T * heads * sizeof(uint2) + sizeof(int);
}

cudaError_t launch_kv4_decode(const Kv4DecodeArgs& a, void* workspace, cudaStream_t s) {
  const kvd::Plan plan = kvd::plan_of(a.B, a.T, a.max_len, a.heads, a.kv, a.hd);
  if (plan.places >> 32) return cudaErrorInvalidValue;  // a workspace of a terabyte
  kvd::Args p;
  p.a = a;
  p.hc = plan.hc;
  p.q_min = plan.q_min;
  p.split = (uint32_t)plan.split;
  p.ws_o = (float*)workspace;
  p.ws_ml = (float2*)(p.ws_o + plan.places * a.hd);
  p.ws_n = (uint2*)(p.ws_ml + plan.places);
  p.ws_falls = (int*)(p.ws_n + (size_t)a.T * a.heads);
  if (a.hd == 256) return plan.nt == 1 ? kvd::run<256, 1>(p, plan, s) : kvd::run<256, 2>(p, plan, s);
  if (a.hd == 128) return plan.nt == 1 ? kvd::run<128, 1>(p, plan, s) : plan.nt == 2 ? kvd::run<128, 2>(p, plan, s) : kvd::run<128, 4>(p, plan, s);
  return plan.nt == 1 ? kvd::run<64, 1>(p, plan, s) : plan.nt == 2 ? kvd::run<64, 2>(p, plan, s) : kvd::run<64, 4>(p, plan, s);
}
