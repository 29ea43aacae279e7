// Attention of one new token per sequence over the 8-bit paged cache (kv8.cuh):
//
//   o = sum_j softmax_j(scale q . k_j) v_j,   k_j = code * k_scale[page, head],  v_j = code * v_scale[page, head]
//
// Bound by the cache's bytes: 2 D bytes a token and key head for 4 G D operations (G query heads share a key head).  Measured, with
// 32 query and 8 key heads of 128: 131067 tokens of one sequence 54.1 us (268 MB: 5.3 TB/s in the main kernel), 128 sequences of up to
// 8192 tokens 50.7 us; 64 sequences of 1024 tokens with 28 and 4 heads 22.4 us, of which 4 us pass before the first codes are
// there and 4 us in the join.
//
// A warp takes 16 tokens a step.  Each warp has a queue of steps in shared memory that its first lane keeps filled by TMA, a few
// steps ahead; no warp waits for another one, so rows of any length run side by side.  A lane reads its codes from the
// (swizzled, so free of bank conflicts at head dims 128 and 256) tile in the order that the matrix instruction (16 x 8 x 16,
// fp16 in, fp32 sums) wants its operands, and makes fp16 of them, exactly.
//   S = Q K^T   A = Q (heads as rows), B = K: the lane (g, t) holds quarter t of token g's row.  Which dimension stands at which
//               place of the sum is free, so a lane's dimensions are whatever its loads bring.
//   O^T = V^T P^T   A = V^T, B = P: the probabilities are already where the B operand wants them (the 2t-th and 2t+1-th token of
//               head g), and the lane (g, t) holds dimensions of unit g for those tokens, whose bytes are interleaved in pairs.
// Queries are brought within fp16 by a power of two per row (exact for bf16 and fp16 but for values 2^24 below the row's
// largest).
//
// Page scales.  k_scale multiplies the scores.  v_scale goes into the exponent: w_j = exp2(s_j + log2 v_scale - m) with m the
// running maximum of that sum, less KA_BELOW, so that weights stay within fp16 whatever the pages' scales, and the softmax's
// denominator is sum w_j / v_scale.  m moves only when a weight would pass 2^15; then the largest is 2^KA_BELOW.  A weight is rounded
// once, to fp16: by 2^-11 of it, or below fp16's normal numbers by 2^-32 of the largest.
//
// Work: the steps of all rows (sequence, key head, head tile) are one list that is dealt to the warps in equal runs, so any mix
// of lengths fills the GPU; a row counts KA_ROW steps more than it has, the cost of beginning one.  A warp that has all steps of
// a row writes its output.  Else it leaves (m, l, o); where all of a block's runs lie in one row, the block joins its warps'
// first and leaves one.  The warp that has a row's first step says which row it is, for kv8_attn_join_kernel, which adds a
// row's parts in the order of the warps.  No atomics: results do not depend on timing.
//
// Where there are no more rows than SMs and the block table has room for few steps a warp only (kv8_attn_alone), each row gets a
// block of its own instead (by_row): no list of all rows, no parts, no second kernel.  One sequence of 211 tokens with 14 and 2
// heads of 64 takes 6.4 us so, 10.2 us from the list.
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace trlb {

enum { SITE_KV8_ATTN = 1410 };

constexpr int KA_STEP = 16;          // tokens of a warp's step
constexpr int KA_ROW = 4;            // steps that a row's beginning is worth
constexpr int KA_JOIN = 512;         // threads of a joining block: 22.7 us for 64 x 1024 tokens, with 256 threads 24.2
constexpr int KA_MAX_SEQS = 4096;    // the prefix sums of their steps stand in shared memory
constexpr float KA_NONE = -3.4028234663852886e38f;  // maximum of no token: no score is below it, and exp2(-inf - m) is 0
constexpr float KA_BELOW = 7.f;      // a weight is at most 2^15 before m moves, and the largest 2^7 when it has

// One block an SM, with as many warps as registers allow, and the steps in a warp's queue: about 190 KB of codes under way.
__host__ __device__ constexpr int kv8_attn_warps(int D, int HT) { return D == 256 ? 8 : (D == 64 && HT == 8 ? 16 : 12); }
__host__ __device__ constexpr int kv8_attn_stages(int D) { return D == 256 ? 3 : (D == 128 ? 4 : (D == 96 ? 5 : 6)); }
// Steps of a warp up to which a block takes a row alone: 4 sequences with 28 and 4 heads of 128 take 10.0 us alone and 11.7 from
// the list at 700 tokens, 11.8 and 12.9 at 1000, 13.9 and 13.2 at 1500; with 8 heads of 256 11.9 and 13.8 at 400, 15.1 and 13.4 at 700.
__host__ __device__ constexpr int kv8_attn_alone(int D) { return D == 256 ? 3 : 5; }
// Swizzle of a row's bytes in shared memory; 96 bytes stand as they are.
__host__ __device__ constexpr int kv8_attn_swizzle(int D) { return D % 128 == 0 ? 128 : (D == 64 ? 64 : 0); }

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) { return unpack_bf16(u); }
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float x) { *p = __float2bfloat16(x); }
__device__ __forceinline__ void store1(__half* p, float x) { *p = __float2half(x); }

template <int BYTES>
__device__ __forceinline__ void read_codes(uint32_t* w, uint32_t src) {
  if constexpr (BYTES == 16) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(src) : "memory");
  else if constexpr (BYTES == 8) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(src) : "memory");
  else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(src) : "memory");
}
// Address of byte x of row r in a tile of 16 rows of D bytes as TMA leaves it.
template <int D>
__device__ __forceinline__ uint32_t tile_at(int r, int x) {
  if constexpr (D % 128 == 0) return (x >> 7) * 2048 + r * 128 + ((x & 127) ^ ((r & 7) << 4));
  else if constexpr (D == 64) return r * 64 + (x ^ (((r >> 1) & 3) << 4));
  else return r * D + x;
}
// The token of a step at place c of eight: an order in which lanes that read together read different banks.
template <int D>
__device__ __forceinline__ int place(int c) { return D % 128 == 0 ? (c >> 1) | ((c & 1) << 2) : c; }

__device__ __forceinline__ uint32_t pack_out(float a, float b, __nv_bfloat16) { return pack_bf16(a, b); }
__device__ __forceinline__ uint32_t pack_out(float a, float b, __half) { return pack_f16(a, b); }

struct alignas(16) SharedRow {
  int seq, head, heads;  // seq < 0: none
  int last;              // warp of the last step
  int joined0, joined1;  // blocks whose warps' parts are one, at the first warp's place
  int pad[2];
};

struct Kv8AttnArgs {
  CUtensorMap k, v;  // codes as [pages * heads][page size][D], boxes of 16 rows
  const void* q;
  long long q_row, q_head;
  const float *k_scale, *v_scale;
  const int *table, *seq_lens, *slots;
  void* out;
  float* part;      // [2 * warps][HT][D]: sums of the row that began before a warp's run, of the row that ends behind it
  float2* part_ml;  // [2 * warps][HT]: their maxima and denominators
  SharedRow* rows;  // [warps]: the row whose first step is in a warp's run and whose last is not
  int* status;
  int pages, Hk, G, tiles, page_shift, table_rows, max_blocks, B, window, by_row;
  float scale;
};

// Steps of a sequence and where they begin.  seq_lens holds the newest token's position: tokens 0 .. seq_len are seen.
// A slot that the table does not have, and tokens beyond a row of the table, are reported and count for nothing.
__device__ __forceinline__ int kv8_steps(const Kv8AttnArgs& a, int b, int& lo, int& hi) {
  const int slot = a.slots ? a.slots[b] : b;
  hi = lo = 0;
  if (slot < 0 || slot >= a.table_rows) {
    report_error(a.status, ERR_BOUNDS, SITE_KV8_ATTN, slot);
    return 0;
  }
  const int newest = a.seq_lens[slot];
  if (newest < 0) return 0;
  const long long cap = (long long)a.max_blocks << a.page_shift;
  if (newest >= cap) report_error(a.status, ERR_BOUNDS, SITE_KV8_ATTN, newest);
  hi = (int)min((long long)newest + 1, cap);
  lo = a.window > 0 ? max(0, hi - a.window) : 0;
  return (hi + KA_STEP - 1) / KA_STEP - lo / KA_STEP;
}

// prefix[b] = cost of one row of each of the sequences before b, prefix[B] = of all
template <int WARPS>
__device__ __forceinline__ void kv8_prefix(const Kv8AttnArgs& a, int* prefix, int* warp_sums) {
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int per = (a.B + WARPS * 32 - 1) / (WARPS * 32), i0 = min(a.B, tid * per), i1 = min(a.B, i0 + per);
  int sum = 0, last = 0, lo, hi;
  for (int i = i0; i < i1; ++i) {
    const int n = kv8_steps(a, i, lo, hi);
    last = n > 0 ? n + KA_ROW : 0;
    sum += last;
  }
  int run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += x;
  }
  if (lane == 31) warp_sums[wid] = run;
  __syncthreads();
  int before = run - sum;
  for (int w = 0; w < wid; ++w) before += warp_sums[w];
  for (int i = i0; i < i1; ++i) {
    prefix[i] = before;
    if (per > 1) {
      const int n = kv8_steps(a, i, lo, hi);
      last = n > 0 ? n + KA_ROW : 0;
    }
    before += last;
  }
  if (tid == WARPS * 32 - 1) prefix[a.B] = before;
  __syncthreads();
}
// Quotient of numbers that mostly fit into 32 bits.
__device__ __forceinline__ int kv8_div(long long x, int d) {
  return (x >> 31) == 0 ? (int)((unsigned)x / (unsigned)d) : (int)(x / d);
}

template <int D, int HT, typename T>
__global__ void __launch_bounds__(kv8_attn_warps(D, HT) * 32, 1)
kv8_attn_kernel(const __grid_constant__ Kv8AttnArgs a) {
  constexpr int KU = D % 64 == 0 ? 16 : 8, KN = D / (4 * KU);                         // K: bytes of a lane's unit, units a row
  constexpr int VU = D % 128 == 0 ? 16 : (D % 64 == 0 ? 8 : 4), VN = D / (8 * VU);    // V: the same
  constexpr int KW = D / 16, VW = D / 32;                                             // words of a row in a lane
  constexpr int KA_WARPS = kv8_attn_warps(D, HT), KA_THREADS = KA_WARPS * 32;
  constexpr int NT = HT / 8, S = kv8_attn_stages(D), STAGE = 32 * D, BOX = D % 128 == 0 ? 128 : D;
  extern __shared__ uint8_t smem_raw[];  // [warps][S][K tile, V tile] on 1024 bytes, then prefix [B + 1]
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  int* prefix = reinterpret_cast<int*>(smem + KA_WARPS * S * STAGE);
  __shared__ uint64_t full[KA_WARPS][S];
  __shared__ int abort_flag;
  __shared__ float2 sh_ml[KA_WARPS][HT];
  __shared__ int4 sh_row;
  __shared__ int warp_sums[KA_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < S; ++i) mbar_init(&full[wid][i], 1);
    mbar_fence_init();
    if (wid == 0) {
      abort_flag = 0;
      tma_prefetch_desc(&a.k);
      tma_prefetch_desc(&a.v);
    }
  }
  pdl_launch_dependents();
  pdl_wait();
  const int rows_per_seq = a.Hk * a.tiles, warp = blockIdx.x * KA_WARPS + wid;
  long long total, run, u0, u1, block0, block1;
  int b = 0;
  bool joined = false;  // all of the block's runs lie in one row
  SharedRow shared = {-1, 0, 0, 0, 0, 0, {0, 0}};
  if (a.by_row) {
    b = blockIdx.x / rows_per_seq;
    const int row = blockIdx.x % rows_per_seq;
    if (tid == 0) {  // the row's sequence is all of the list
      int lo, hi;
      const int n = kv8_steps(a, b, lo, hi);
      prefix[b] = 0;
      prefix[b + 1] = n > 0 ? n + KA_ROW : 0;
    }
    __syncthreads();  // shows the mbarriers, too
    const int cost = prefix[b + 1];
    if (cost == 0) {
      const int h0 = (row % a.tiles) * HT, heads = min(HT, a.G - h0);
      for (int i = tid; i < heads * D; i += KA_THREADS)
        store1(reinterpret_cast<T*>(a.out) + ((size_t)b * a.Hk * a.G + row / a.tiles * a.G + h0) * D + i, 0.f);
      return;
    }
    total = (long long)cost * rows_per_seq;
    run = (cost - KA_ROW + KA_WARPS - 1) / KA_WARPS;
    block0 = (long long)row * cost + KA_ROW;
    block1 = (long long)(row + 1) * cost;
    u0 = min(block1, block0 + wid * run);
    u1 = min(block1, u0 + run);
    joined = true;
  } else {
    kv8_prefix<KA_WARPS>(a, prefix, warp_sums);  // its barriers show the mbarriers, too
    // sequences without a token to see have no steps: their zeros are written here
    for (int b = blockIdx.x; b < a.B; b += gridDim.x)
      if (prefix[b + 1] == prefix[b])
        for (int i = tid; i < a.Hk * a.G * D; i += KA_THREADS)
          store1(reinterpret_cast<T*>(a.out) + (size_t)b * a.Hk * a.G * D + i, 0.f);
    const long long warps = (long long)gridDim.x * KA_WARPS;
    total = (long long)prefix[a.B] * rows_per_seq;
    run = max(1ll, (total + warps - 1) / warps);
    u0 = (long long)warp * run;
    u1 = min(total, u0 + run);
    block0 = (long long)blockIdx.x * KA_WARPS * run;
    block1 = min(total, block0 + KA_WARPS * run);
    if (block0 < block1) {  // the sequence that the block begins in
      int hi = a.B - 1;
      while (b < hi) {
        const int mid = (b + hi + 1) >> 1;
        if ((long long)prefix[mid] * rows_per_seq <= block0) b = mid; else hi = mid - 1;
      }
      const int cost = prefix[b + 1] - prefix[b];
      const long long seq0 = (long long)prefix[b] * rows_per_seq;
      joined = seq0 + (long long)(kv8_div(block0 - seq0, cost) + 1) * cost >= block1;
    }
  }
  if (lane < HT) sh_ml[wid][lane] = make_float2(KA_NONE, 0.f);
  uint8_t* queue = smem + wid * S * STAGE;
  int slot_in = 0, slot_out = 0;
  uint32_t parity = 0;
  // of the block's row, where its warps join
  int join_seq = 0, join_head = 0, join_heads = 0;
  bool join_whole = false;
  size_t join_part = 0;
  for (long long u = u0; u < u1;) {
    while (prefix[b + 1] == prefix[b] || (long long)prefix[b + 1] * rows_per_seq <= u) ++b;
    const int cost = prefix[b + 1] - prefix[b], steps = cost - KA_ROW;
    const long long seq0 = (long long)prefix[b] * rows_per_seq;
    const int row = kv8_div(u - seq0, cost);
    const long long row0 = seq0 + (long long)row * cost;  // its beginning counts first, then its steps
    const int s0 = (int)max(0ll, u - row0 - KA_ROW), s1 = (int)min((long long)steps, u1 - row0 - KA_ROW);
    const int kvh = row / a.tiles, h0 = (row % a.tiles) * HT, heads = min(HT, a.G - h0);
    const bool begins = joined ? block0 - row0 <= KA_ROW : s0 == 0;  // the row's first step is in the run (of the block)
    const bool whole = begins && row0 + cost <= (joined ? block1 : u1);
    if (begins && !whole && (joined ? wid == 0 : s1 > 0)) {
      const long long per = KA_WARPS * run;
      // blocks that lie in the row; the list's last one may be shorter than the others
      const long long end = row0 + cost >= total ? total + per - 1 : row0 + cost;
      shared = {b, kvh * a.G + h0, heads, (int)((row0 + cost - 1) / run), (int)((row0 + per - 1) / per), (int)(end / per), {0, 0}};
    }
    join_seq = b;
    join_head = kvh * a.G + h0;
    join_heads = heads;
    join_whole = whole;
    join_part = (size_t)2 * blockIdx.x * KA_WARPS + (begins ? 1 : 0);
    u = row0 + cost;
    if (s1 <= s0) continue;  // no more of it than its beginning
    int tok_lo, tok_hi;
    kv8_steps(a, b, tok_lo, tok_hi);
    const int slot = a.slots ? a.slots[b] : b;
    const int base = tok_lo / KA_STEP;  // step s covers the tokens (base + s) * 16 ...
    const int* table = a.table + (size_t)slot * a.max_blocks;
    const int per_page = a.page_shift - 4;  // log2 of the steps of a page
    const int page_first = (base + s0) >> per_page, page_last = (base + s1 - 1) >> per_page;

    // Pages, 32 at a time, one a lane: those that loads are taken from and the ones behind them, and the scales of those that
    // are computed with and of the ones behind them.
    auto pages_from = [&](int first) {
      int blk = -1;
      if (first + lane <= page_last) {
        blk = table[first + lane];
        if (blk < 0 || blk >= a.pages) {  // not a page of the cache: its tokens count for nothing
          report_error(a.status, ERR_BOUNDS, SITE_KV8_ATTN, blk);
          blk = -1;
        }
      }
      return blk;
    };
    auto scales_of = [&](int blk, float& k, float& v) {
      k = v = 0.f;
      if (blk >= 0) {
        k = a.k_scale[(size_t)blk * a.Hk + kvh];
        v = a.v_scale[(size_t)blk * a.Hk + kvh];
      }
    };
    int load_from = page_first, pages = pages_from(page_first), pages_next = page_last - page_first >= 32 ? pages_from(page_first + 32) : -1;
    float ks, vs, ks_next = 0.f, vs_next = 0.f;
    int scale_from = page_first;
    scales_of(pages, ks, vs);
    int next = s0;
    auto copy = [&]() {  // the codes of step `next` into the queue
      if (next >= s1) return;
      const int page = (base + next) >> per_page;
      if (page - load_from >= 32) {
        load_from += 32;
        pages = pages_next;
        scales_of(pages, ks_next, vs_next);
        pages_next = pages_from(load_from + 32);
      }
      const int blk = __shfl_sync(0xffffffffu, pages, page - load_from);  // every lane is here: the slot has been read
      if (lane == 0) {
        uint64_t* bar = &full[wid][slot_in];
        if (blk < 0) {
          mbar_arrive(bar);  // nothing to read; the step has no weight
        } else {
          uint8_t* dst = queue + slot_in * STAGE;
          const int y = ((base + next) & ((1 << per_page) - 1)) << 4, z = blk * a.Hk + kvh;
          mbar_expect_tx(bar, STAGE);
#pragma unroll
          for (int i = 0; i < D / BOX; ++i) {
            tma_load_3d(dst + i * 16 * BOX, &a.k, bar, i * BOX, y, z);
            tma_load_3d(dst + 16 * D + i * 16 * BOX, &a.v, bar, i * BOX, y, z);
          }
        }
      }
      ++next;
      slot_in = slot_in + 1 == S ? 0 : slot_in + 1;
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) copy();

    // Queries of this row: heads g (and g + 8) as A operands, brought to at most 2 in magnitude.
    uint32_t qa[KW][2 * NT];
    float cq[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = g + 8 * n;
      const T* qp = reinterpret_cast<const T*>(a.q) + (long long)b * a.q_row + (long long)(kvh * a.G + h0 + h) * a.q_head;
      uint32_t most = 0;  // the largest magnitude's bits: those of infinities and NaN are above all others
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const int d = KU * (t + 4 * (w / (KU / 4))) + 4 * (w % (KU / 4));
        const uint2 raw = h < heads ? *reinterpret_cast<const uint2*>(qp + d) : make_uint2(0, 0);
        qa[w][2 * n] = raw.x;
        qa[w][2 * n + 1] = raw.y;
        const float2 x = unpack2<T>(raw.x), y = unpack2<T>(raw.y);
        auto bits = [](float f) { return __float_as_uint(f) & 0x7fffffffu; };
        most = max(max(most, max(bits(x.x), bits(x.y))), max(bits(y.x), bits(y.y)));
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int e = min(120, max(-100, (int)(most >> 23) - 127));
      const float inv = kv8_pow2(-e);
      // a query that is not finite has NaN as its output: its scores are infinite or NaN, all of them
      cq[n] = most < 0x7f800000u ? a.scale * 1.4426950408889634f * kv8_pow2(e) : NAN;
#pragma unroll
      for (int w = 0; w < KW; ++w)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 x = unpack2<T>(qa[w][2 * n + i]);
          qa[w][2 * n + i] = pack_f16(x.x * inv, x.y * inv);
        }
    }
    float m[NT], l[NT], o[2 * VW][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = KA_NONE;
      l[n] = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * VW; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][n][k] = 0.f;
    }

    int page_now = -1;
    float kscale = 0.f, lv = 0.f, inv_v = 0.f;
    int s = s0;
    for (; s < s1; ++s) {
      copy();
      if (!mbar_wait(&full[wid][slot_out], parity, &abort_flag, a.status, SITE_KV8_ATTN)) break;
      const uint32_t kq = smem_u32(queue) + slot_out * STAGE, vq = kq + 16 * D;
      if (++slot_out == S) {
        slot_out = 0;
        parity ^= 1;
      }
      float sc[2][4];  // scores of the tokens 0-7 and 8-15: [head g: places 2t, 2t + 1][head g + 8: the same]
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t k[KW];
#pragma unroll
        for (int j = 0; j < KN; ++j) read_codes<KU>(k + j * (KU / 4), kq + tile_at<D>(8 * r + place<D>(g), KU * (t + 4 * j)));
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[r][i] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w)
          mma_f16(sc[r], qa[w][0], NT == 2 ? qa[w][2 * (NT - 1)] : 0u, qa[w][1], NT == 2 ? qa[w][2 * (NT - 1) + 1] : 0u,
                  kv8_decode2(k[w]), kv8_decode2_hi(k[w]));
      }
      uint32_t v[4 * VW];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VN; ++j)
          read_codes<VU>(v + r * VW + j * (VU / 4), vq + tile_at<D>((r >> 1) * 8 + place<D>(2 * t + (r & 1)), VU * (place<D>(g) + 8 * j)));
      const int page = (base + s) >> per_page;
      if (page != page_now) {
        page_now = page;
        if (page - scale_from >= 32) {
          scale_from += 32;
          ks = ks_next;
          vs = vs_next;
        }
        kscale = __shfl_sync(0xffffffffu, ks, page - scale_from);
        const float vscale = __shfl_sync(0xffffffffu, vs, page - scale_from);
        lv = __log2f(vscale);  // of a power of two; of 0, where no page is: -inf, no weight
        inv_v = vscale > 0.f ? __frcp_rn(vscale) : 0.f;
      }
      const int tok = (base + s) * KA_STEP;
      const bool edge = tok < tok_lo || tok + KA_STEP > tok_hi || inv_v == 0.f;
      auto hidden = [&](int r) {
        const int x = tok + (r >> 1) * 8 + place<D>(2 * t + (r & 1));
        return x < tok_lo || x >= tok_hi || inv_v == 0.f;
      };
      if (edge) {  // tokens out of sight: what stands there may be anything, NaN included
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (hidden(r))
#pragma unroll
            for (int i = 0; i < VW; ++i) v[r * VW + i] = 0;
      }
      uint32_t p[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float c = cq[n] * kscale;
        float x[4] = {fmaf(sc[0][2 * n], c, lv), fmaf(sc[0][2 * n + 1], c, lv), fmaf(sc[1][2 * n], c, lv), fmaf(sc[1][2 * n + 1], c, lv)};
        if (edge) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (hidden(r)) x[r] = -INFINITY;
        }
        const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        if (__any_sync(0xffffffffu, top > m[n] + 15.f)) {
          float mx = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          mx = fmaxf(m[n], fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) - KA_BELOW);
          const float down = fast_exp2(m[n] - mx);
          m[n] = mx;
          l[n] *= down;
          const float d0 = __shfl_sync(0xffffffffu, down, 8 * t), d1 = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
          for (int i = 0; i < 2 * VW; ++i) {
            o[i][n][0] *= d0;
            o[i][n][1] *= d1;
            o[i][n][2] *= d0;
            o[i][n][3] *= d1;
          }
        }
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = fast_exp2(x[r] - m[n]);
        l[n] = fmaf((w[0] + w[1]) + (w[2] + w[3]), inv_v, l[n]);
        p[n][0] = pack_f16(w[0], w[1]);
        p[n][1] = pack_f16(w[2], w[3]);
      }
#pragma unroll
      for (int i = 0; i < VW; ++i) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t ab = __byte_perm(v[i], v[VW + i], half ? 0x7362 : 0x5140);
          const uint32_t cd = __byte_perm(v[2 * VW + i], v[3 * VW + i], half ? 0x7362 : 0x5140);
          const uint32_t a0 = kv8_decode2(ab), a1 = kv8_decode2_hi(ab), a2 = kv8_decode2(cd), a3 = kv8_decode2_hi(cd);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(o[2 * i + half][n], a0, a1, a2, a3, p[n][0], p[n][1]);
        }
      }
    }
    if (s < s1) {  // a wait has run out (reported): no more copies, and those under way are waited for, with a limit
      for (; s < next; ++s) {
        for (int i = 0; i < 1 << 16 && !mbar_try_wait(&full[wid][slot_out], parity); ++i) {}
        if (++slot_out == S) {
          slot_out = 0;
          parity ^= 1;
        }
      }
      u = u1;
    }

    // o[2 i + half][n]: dimensions 4 i' + 2 half of the lane's units, for the heads 2t ([0], [2]) and 2t + 1 ([1], [3])
    const size_t part = (size_t)2 * warp + (s0 > 0 ? 0 : 1);
    const bool finish = whole && !joined;
    T* out = reinterpret_cast<T*>(a.out) + ((size_t)b * a.Hk * a.G + kvh * a.G + h0) * D;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
      if (t == 0) {
        if (joined) sh_ml[wid][8 * n + g] = make_float2(m[n], l[n]);
        else if (!whole && 8 * n + g < heads) a.part_ml[part * HT + 8 * n + g] = make_float2(m[n], l[n]);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float den = __shfl_sync(0xffffffffu, l[n], 8 * t + 4 * c), inv = den != 0.f ? 1.f / den : 0.f;
        const int h = 8 * n + 2 * t + c;
        if (h >= heads) continue;
        float* keep = joined ? reinterpret_cast<float*>(queue) + h * D : a.part + (part * HT + h) * D;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const int d = VU * (place<D>(g) + 8 * (i / (VU / 4))) + 4 * (i % (VU / 4));
          const float x0 = o[2 * i][n][c], x1 = o[2 * i][n][2 + c], x2 = o[2 * i + 1][n][c], x3 = o[2 * i + 1][n][2 + c];
          if (finish) *reinterpret_cast<uint2*>(out + h * D + d) = make_uint2(pack_out(x0 * inv, x1 * inv, T()), pack_out(x2 * inv, x3 * inv, T()));
          else *reinterpret_cast<float4*>(keep + d) = make_float4(x0, x1, x2, x3);
        }
      }
    }
  }
  if (lane == 0 && !a.by_row) a.rows[warp] = shared;
  if (!joined) return;
  __syncthreads();  // each warp's sums stand in its queue, which is empty
  // (a warp behind the end of the list has seen no row)
  if (wid == 0 && lane == 0) sh_row = make_int4(join_seq, join_head, join_heads, (join_whole ? 2 : 0) + (int)(join_part & 1));
  __syncthreads();
  const int4 jr = sh_row;
  const int heads = jr.z;
  const size_t part = (size_t)2 * blockIdx.x * KA_WARPS + (jr.w & 1);
  for (int i = tid; i < heads * (D / 4); i += KA_THREADS) {
    const int h = i / (D / 4), d = (i % (D / 4)) * 4;
    float mx = sh_ml[0][h].x, den = 0.f;
#pragma unroll
    for (int w = 1; w < KA_WARPS; ++w) mx = fmaxf(mx, sh_ml[w][h].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < KA_WARPS; ++w) {
      const float2 ml = sh_ml[w][h];
      if (ml.x == KA_NONE && ml.y == 0.f) continue;  // a warp without steps has written no sums (one that saw NaN alone has)
      const float f = fast_exp2(ml.x - mx);
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * S * STAGE) + h * D + d);
      den = fmaf(ml.y, f, den);
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
    }
    if (jr.w & 2) {
      const float inv = den != 0.f ? 1.f / den : 0.f;
      T* out = reinterpret_cast<T*>(a.out) + ((size_t)jr.x * a.Hk * a.G + jr.y + h) * D;
      *reinterpret_cast<uint2*>(out + d) = make_uint2(pack_out(acc.x * inv, acc.y * inv, T()), pack_out(acc.z * inv, acc.w * inv, T()));
    } else {
      *reinterpret_cast<float4*>(a.part + (part * HT + h) * D + d) = acc;
      if (d == 0) a.part_ml[part * HT + h] = make_float2(mx, den);
    }
  }
}

// Rows that several warps share: their parts in order.  One block per block of the attention kernel, for the rows that its
// warps began.  A joining warp takes a run of the parts of one head; runs of one head are joined in their order.
template <int D, int HT, typename T>
__global__ void __launch_bounds__(KA_JOIN)
kv8_attn_join_kernel(const __grid_constant__ Kv8AttnArgs a) {
  constexpr int KA_WARPS = kv8_attn_warps(D, HT), E = D / 32, WARPS = KA_JOIN / 32, AHEAD = 8;  // E: a lane's dimensions
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  __shared__ float sh_o[WARPS][D];
  __shared__ float2 sh_ml[WARPS];
  __shared__ SharedRow sh_rows[KA_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  if (threadIdx.x < KA_WARPS * 2) reinterpret_cast<int4*>(sh_rows)[threadIdx.x] = reinterpret_cast<const int4*>(a.rows + blockIdx.x * KA_WARPS)[threadIdx.x];
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int i = 0; i < KA_WARPS; ++i) n += sh_rows[i].seq >= 0;
  if (n == 0) return;
  const int tile = min(HT, a.G), runs = max(1, WARPS / (n * tile));  // warps a head
  for (int x = wid; x < n * tile * runs; x += WARPS) {
    const int h = x / runs % tile;
    int c0 = -1, k = x / runs / tile;
    for (int i = 0; i < KA_WARPS; ++i)
      if (sh_rows[i].seq >= 0 && k-- == 0) c0 = i;
    const SharedRow r = sh_rows[c0];
    if (h >= r.heads) continue;
    c0 += blockIdx.x * KA_WARPS;
    // parts that count: the warps c0 .. j0 - 1, the first one of each joined block up to j1, and the warps from there on
    const int j0 = r.joined0 * KA_WARPS, j1 = r.joined1 * KA_WARPS;
    const bool any = j1 > j0;
    const int n0 = any ? j0 - c0 : 0, n1 = any ? n0 + r.joined1 - r.joined0 : 0;
    const int parts = any ? n1 + max(0, r.last - j1 + 1) : r.last - c0 + 1;
    const int len = (parts + runs - 1) / runs, p0 = (x % runs) * len, p1 = min(parts, p0 + len);
    auto at = [&](int p) {
      const int w = !any || p < n0 ? c0 + p : (p < n1 ? j0 + (p - n0) * KA_WARPS : j1 + (p - n1));
      return ((size_t)2 * w + (p == 0 ? 1 : 0)) * HT + h;
    };
    float m = KA_NONE, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int p = p0; p < p1; p += AHEAD) {  // AHEAD parts under way at once
      float2 ml[AHEAD];
      float y[AHEAD][E], top = m;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        ml[i] = make_float2(KA_NONE, 0.f);
        if (p + i < p1) {
          const size_t q = at(p + i);
          ml[i] = a.part_ml[q];
#pragma unroll
          for (int e = 0; e < E; ++e) y[i][e] = a.part[q * D + lane + 32 * e];
        }
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, ml[i].x);
      const float down = fast_exp2(m - top);
      m = top;
      l *= down;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= down;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (p + i < p1) {
          const float f = fast_exp2(ml[i].x - top);
          l = fmaf(ml[i].y, f, l);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = fmaf(y[i][e], f, o[e]);
        }
    }
    if (runs == 1) {
      const float inv = l != 0.f ? 1.f / l : 0.f;
      T* out = reinterpret_cast<T*>(a.out) + ((size_t)r.seq * a.Hk * a.G + r.head + h) * D;
#pragma unroll
      for (int e = 0; e < E; ++e) store1(out + lane + 32 * e, o[e] * inv);
    } else {  // then no warp takes a second run
#pragma unroll
      for (int e = 0; e < E; ++e) sh_o[wid][lane + 32 * e] = o[e];
      if (lane == 0) sh_ml[wid] = make_float2(m, l);
    }
  }
  if (runs == 1) return;
  __syncthreads();
  if (wid >= n * tile) return;
  const int h = wid % tile, w0 = wid * runs;  // the warps that had this head
  int c0 = -1, k = wid / tile;
  for (int i = 0; i < KA_WARPS; ++i)
    if (sh_rows[i].seq >= 0 && k-- == 0) c0 = i;
  const SharedRow r = sh_rows[c0];
  if (h >= r.heads) return;
  float mx = KA_NONE, den = 0.f, o[E];
  for (int w = w0; w < w0 + runs; ++w) mx = fmaxf(mx, sh_ml[w].x);
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int w = w0; w < w0 + runs; ++w) {
    const float f = fast_exp2(sh_ml[w].x - mx);
    den = fmaf(sh_ml[w].y, f, den);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(sh_o[w][lane + 32 * e], f, o[e]);
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
  T* out = reinterpret_cast<T*>(a.out) + ((size_t)r.seq * a.Hk * a.G + r.head + h) * D;
#pragma unroll
  for (int e = 0; e < E; ++e) store1(out + lane + 32 * e, o[e] * inv);
}

// The most steps that a sequence can have, by the room in its row of the block table and the window.
inline long long kv8_room_steps(long long tokens, long long window) {
  return (window > 0 && window + KA_STEP < tokens ? window + KA_STEP : tokens) / KA_STEP + 1;
}
// Whether each row gets a block: a rule on what the host knows.
inline bool kv8_by_row(int D, int ht, long long rows, long long tokens, long long window) {
  return rows <= trlb_host::sm_count() && kv8_room_steps(tokens, window) <= (long long)kv8_attn_alone(D) * kv8_attn_warps(D, ht);
}
inline int kv8_head_tile(int D, int G) { return G <= 8 || D > 128 ? 8 : 16; }

template <int D, int HT, typename T>
int kv8_attn_launch(Kv8AttnArgs& a, const void* k, const void* v, cudaStream_t st) {
  constexpr int WARPS = kv8_attn_warps(D, HT);
  const size_t queues = (size_t)WARPS * kv8_attn_stages(D) * 32 * D + 1024, smem = queues + (size_t)(a.B + 1) * 4;
  static bool ready[64] = {};  // per device; a second thread that sets it at once sets the same
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !ready[dev]) {
    e = cudaFuncSetAttribute(kv8_attn_kernel<D, HT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)queues + (KA_MAX_SEQS + 1) * 4);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) ready[dev] = true;
  }
  const uint64_t tiles = (uint64_t)a.pages * a.Hk, page = 1ull << a.page_shift;
  const uint32_t box = D % 128 == 0 ? 128 : D;
  if (trlb_host::make_tmap_3d_u8(&a.k, k, D, page, tiles, box, KA_STEP, kv8_attn_swizzle(D)) ||
      trlb_host::make_tmap_3d_u8(&a.v, v, D, page, tiles, box, KA_STEP, kv8_attn_swizzle(D)))
    return -6;
  const int blocks = a.by_row ? a.B * a.Hk * a.tiles : trlb_host::sm_count();
  a.part_ml = reinterpret_cast<float2*>(a.part + (size_t)2 * blocks * WARPS * HT * D);  // each on 16 bytes
  a.rows = reinterpret_cast<SharedRow*>(a.part_ml + (size_t)2 * blocks * WARPS * HT);
  e = trlb_host::launch_kernel(kv8_attn_kernel<D, HT, T>, dim3(blocks), dim3(WARPS * 32), smem, st, trlb_host::pdl_enabled(), a);
  if (e != cudaSuccess || a.by_row) return (int)e;
  // it waits for the attention kernel by itself, so it may always be set up under that kernel's end
  return (int)trlb_host::launch_kernel(kv8_attn_join_kernel<D, HT, T>, dim3(blocks), dim3(KA_JOIN), 0, st, true, a);
}
template <typename T>
int kv8_attn_pick(Kv8AttnArgs& a, const void* k, const void* v, int D, cudaStream_t st) {
  const int ht = kv8_head_tile(D, a.G);
  a.tiles = (a.G + ht - 1) / ht;
  switch (D) {
    case 64: return ht == 8 ? kv8_attn_launch<64, 8, T>(a, k, v, st) : kv8_attn_launch<64, 16, T>(a, k, v, st);
    case 96: return ht == 8 ? kv8_attn_launch<96, 8, T>(a, k, v, st) : kv8_attn_launch<96, 16, T>(a, k, v, st);
    case 128: return ht == 8 ? kv8_attn_launch<128, 8, T>(a, k, v, st) : kv8_attn_launch<128, 16, T>(a, k, v, st);
    case 256: return kv8_attn_launch<256, 8, T>(a, k, v, st);
  }
  return -1;
}

}  // namespace trlb

using namespace trlb;

// fp32 words of scratch that a call needs: parts of rows that several blocks share.  `tokens`: what a row of the block table has
// room for.  -1: so many steps that the list's 32-bit prefix sums might not hold them.
TRLB_API long long trlb_kv8_attn_scratch(int B, int Hq, int Hk, int D, long long tokens, int window) {
  const int ht = kv8_head_tile(D, Hq / Hk);
  if (kv8_room_steps(tokens, window) + KA_ROW > 2147483647ll / B) return -1;
  if (kv8_by_row(D, ht, (long long)B * Hk * ((Hq / Hk + ht - 1) / ht), tokens, window)) return 0;
  return (2ll * ht * (D + 2) + sizeof(SharedRow) / 4) * kv8_attn_warps(D, ht) * trlb_host::sm_count();
}

// q [B, Hq, D] bf16 (dtype 0) or fp16 (1) with strides in elements (multiples of 4, rows 8 bytes aligned); out dense, on 16
// bytes.  page_size a power of two, 16 or more.  window 0: everything.  Rows with seq_len < 0 get zeros.
struct Kv8AttnCall {
  const void *q, *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  const int *table, *seq_lens, *slots;
  float* part;
  void* out;
  int* status;
  cudaStream_t stream;
  long long q_row, q_head;
  int dtype, pages, page_size, table_rows, max_blocks, B, Hq, Hk, D, window, part_words;
  float scale;
};
TRLB_API int trlb_kv8_decode_attn(const Kv8AttnCall* call) {
  const Kv8AttnCall c = *call;
  if (c.B == 0) return 0;
  if (c.Hk <= 0 || c.Hq <= 0 || c.Hq % c.Hk || c.B > KA_MAX_SEQS || c.window < 0) return -2;
  if (c.page_size < KA_STEP || (c.page_size & (c.page_size - 1))) return -3;
  if ((long long)c.pages * c.Hk > 2147483647ll) return -5;
  int shift = 0;
  while ((1 << shift) < c.page_size) ++shift;
  Kv8AttnArgs a{{}, {}, c.q, c.q_row, c.q_head, c.k_scale, c.v_scale, c.table, c.seq_lens, c.slots, c.out, c.part, nullptr,
                nullptr, c.status, c.pages, c.Hk, c.Hq / c.Hk, 1, shift, c.table_rows, c.max_blocks, c.B, c.window, 0, c.scale};
  const long long words = trlb_kv8_attn_scratch(c.B, c.Hq, c.Hk, c.D, (long long)c.max_blocks << shift, c.window);
  if (words < 0) return -8;
  if (c.part_words < words) return -7;
  a.by_row = words == 0;
  if (c.dtype == 0) return kv8_attn_pick<__nv_bfloat16>(a, c.k_codes, c.v_codes, c.D, c.stream);
  if (c.dtype == 1) return kv8_attn_pick<__half>(a, c.k_codes, c.v_codes, c.D, c.stream);
  return -4;
}
