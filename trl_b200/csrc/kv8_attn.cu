// Attention of one new token per sequence over the 8-bit paged cache (kv8.cuh):
//
//   o = sum_j softmax_j(scale q . k_j) v_j,   k_j = code * k_scale[page, head],  v_j = code * v_scale[page, head]
//
// Bound by the cache's bytes: 2 D bytes a token and key head for 4 G D operations (G query heads share a key head).
//
// A warp takes 16 tokens a step.  Their codes go from memory straight into registers in the order that the matrix
// instruction wants its operands (16 x 8 x 16, fp16 in, fp32 sums): nothing of the cache passes through shared memory and no
// warp waits for another one until the sums are joined.
//   S = Q K^T   A = Q (heads as rows), B = K: the lane (g, t) holds quarter t of token g's row.  Which dimension stands at
//               which place of the sum is free, so a lane's dimensions are whatever its loads bring.
//   O^T = V^T P^T   A = V^T, B = P: the probabilities are already where the B operand wants them (tokens 2t, 2t + 1 of head g),
//               and the lane (g, t) holds dimensions of unit g for the tokens 2t, 2t + 1, 2t + 8, 2t + 9, whose bytes are
//               interleaved in pairs.
// Codes become fp16 exactly.  Queries are brought within fp16 by a power of two per row (exact for bf16 and fp16 but for
// values 2^24 below the row's largest).
//
// Page scales.  k_scale multiplies the scores.  v_scale goes into the exponent: w_j = exp2(s_j + log2 v_scale - m) with m the
// running maximum of that sum, so that weights stay within fp16 whatever the pages' scales, and the softmax's denominator is
// sum w_j / v_scale.  m moves only when a weight would pass 2^8.
//
// Work: the steps of all (sequence, key head, head tile) are one list that is dealt to the blocks in equal runs, so any mix
// of lengths fills the GPU.  A block whose run covers all steps of a row writes its output; else it leaves its (m, l, o) for
// kv8_attn_join_kernel, which adds a row's parts in the order of the blocks.  No atomics: results do not depend on timing.
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace trlb {

enum { SITE_KV8_ATTN = 1410 };

constexpr int KA_WARPS = 4, KA_THREADS = KA_WARPS * 32;
constexpr int KA_STEP = 16;          // tokens of a warp's step
constexpr int KA_MAX_SEQS = 8192;    // the prefix sums of their steps stand in shared memory
constexpr float KA_NONE = -1e30f;    // maximum of no token: finite, so that exp2(-inf - m) is 0

// Blocks an SM holds: what the registers of a thread (codes of two steps, queries, sums) leave room for.
__host__ __device__ constexpr int kv8_attn_per_sm(int D, int HT) { return D * HT > 128 * 8 ? 2 : 3; }

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

// Bytes that are read once: past the first-level cache.
template <int BYTES>
__device__ __forceinline__ void load_codes(uint32_t* w, const uint8_t* p) {
  if constexpr (BYTES == 16) {
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  } else if constexpr (BYTES == 8) {
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
  }
}

struct Kv8AttnArgs {
  const void* q;
  long long q_row, q_head;
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  const int *table, *seq_lens, *slots;
  void* out;
  float* part;  // [2 * blocks][HT][D + 2]
  int *status;
  int pages, Hk, G, tiles, page_shift, table_rows, max_blocks, B, window, min_run;
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

// prefix[b] = steps of the sequences before b, prefix[B] = of all
__device__ __forceinline__ void kv8_prefix(const Kv8AttnArgs& a, int* prefix, int* warp_sums) {
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int per = (a.B + KA_THREADS - 1) / KA_THREADS;
  int sum = 0, lo, hi;
  for (int i = tid * per; i < min(a.B, (tid + 1) * per); ++i) sum += kv8_steps(a, i, lo, hi);
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
  for (int i = tid * per; i < min(a.B, (tid + 1) * per); ++i) {
    prefix[i] = before;
    before += kv8_steps(a, i, lo, hi);
  }
  if (tid == KA_THREADS - 1) prefix[a.B] = before;
  __syncthreads();
}
// Steps a block takes: all of them in equal runs, but no run so short that its warps would have less than a step.
__device__ __forceinline__ long long kv8_run(const Kv8AttnArgs& a, long long total, int blocks) {
  const long long even = (total + blocks - 1) / blocks;
  return even > a.min_run ? even : a.min_run;
}

template <int D, int HT, typename T>
__global__ void __launch_bounds__(KA_THREADS, kv8_attn_per_sm(D, HT))
kv8_attn_kernel(const __grid_constant__ Kv8AttnArgs a) {
  constexpr int KU = D % 64 == 0 ? 16 : 8, KN = D / (4 * KU);                         // K: units of a lane's loads, loads a row
  constexpr int VU = D % 128 == 0 ? 16 : (D % 64 == 0 ? 8 : 4), VN = D / (8 * VU);    // V: the same
  constexpr int KW = D / 16, VW = D / 32;                                             // words of a row in a lane
  constexpr int NT = HT / 8;
  extern __shared__ __align__(16) float smem[];
  float* sh_o = smem;                                  // [warps][HT][D]
  float* sh_m = sh_o + KA_WARPS * HT * D;              // [warps][HT]
  float* sh_l = sh_m + KA_WARPS * HT;
  int* prefix = reinterpret_cast<int*>(sh_l + KA_WARPS * HT);  // [B + 1]
  __shared__ int warp_sums[KA_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  kv8_prefix(a, prefix, warp_sums);
  const int rows_per_seq = a.Hk * a.tiles;
  const long long total = (long long)prefix[a.B] * rows_per_seq, run = kv8_run(a, total, gridDim.x);
  // rows without a token to see have no steps: their zeros are written here
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (prefix[b + 1] == prefix[b])
      for (int i = tid; i < a.Hk * a.G * D; i += KA_THREADS)
        store1(reinterpret_cast<T*>(a.out) + (size_t)b * a.Hk * a.G * D + i, 0.f);
  long long u = (long long)blockIdx.x * run;
  const long long u1 = min(total, u + run);
  const long long first = u;
  int b = 0;
  if (u < u1) {  // the sequence that step u belongs to
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)prefix[mid] * rows_per_seq <= u) lo = mid; else hi = mid - 1;
    }
    b = lo;
    // sequences without steps share their prefix with the next one: the last of equals is the one with steps
  }
  while (u < u1) {
    while (prefix[b + 1] == prefix[b] || (long long)prefix[b + 1] * rows_per_seq <= u) ++b;
    int tok_lo, tok_hi;
    const int steps = kv8_steps(a, b, tok_lo, tok_hi);
    const long long seq_u = u - (long long)prefix[b] * rows_per_seq;
    const int row = (int)(seq_u / steps), s0 = (int)(seq_u % steps);
    const int s1 = (int)min((long long)steps, s0 + (u1 - u));
    const int kvh = row / a.tiles, h0 = (row % a.tiles) * HT, heads = min(HT, a.G - h0);
    const int slot = a.slots ? a.slots[b] : b;
    const int base = tok_lo / KA_STEP;  // step s covers the tokens (base + s) * 16 ...
    const int* table = a.table + (size_t)slot * a.max_blocks;

    uint32_t kw[2][2 * KW], vw[2][4 * VW];
    float ks[2], vs[2];
    const int page_mask = (1 << a.page_shift) - 1;
    auto page_of = [&](int s) {
      return table[((base + s) * KA_STEP) >> a.page_shift];
    };
    auto load = [&](int s, int blk, uint32_t* k, uint32_t* v, float& kscale, float& vscale) {
      if (blk < 0 || blk >= a.pages) {  // not a page of the cache: no token of the step counts
        report_error(a.status, ERR_BOUNDS, SITE_KV8_ATTN, blk);
        vscale = 0.f;
        kscale = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * KW; ++i) k[i] = 0;
#pragma unroll
        for (int i = 0; i < 4 * VW; ++i) v[i] = 0;
        return;
      }
      const size_t tile = (size_t)blk * a.Hk + kvh;
      const size_t at = ((tile << a.page_shift) + (((base + s) * KA_STEP) & page_mask)) * D;
      const uint8_t* kp = a.k + at + (size_t)g * D + t * KU;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < KN; ++j) load_codes<KU>(k + r * KW + j * (KU / 4), kp + r * 8 * D + j * 4 * KU);
      const uint8_t* vp = a.v + at + (size_t)(2 * t) * D + g * VU;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VN; ++j) load_codes<VU>(v + r * VW + j * (VU / 4), vp + ((r >> 1) * 8 + (r & 1)) * D + j * 8 * VU);
      kscale = a.k_scale[tile];
      vscale = a.v_scale[tile];
    };

    int s = s0 + wid;
    int blk_next = 0;
    if (s < s1) {
      const int blk = page_of(s);
      if (s + KA_WARPS < s1) blk_next = page_of(s + KA_WARPS);
      load(s, blk, kw[0], vw[0], ks[0], vs[0]);
    }
    // queries of this row tile: rows g (and g + 8) as A operands, brought to at most 2 in magnitude
    uint32_t qa[KW][2 * NT];
    float cq[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = g + 8 * n;
      const T* qp = reinterpret_cast<const T*>(a.q) + (long long)b * a.q_row + (long long)(kvh * a.G + h0 + h) * a.q_head;
      uint2 raw[KW];
      float most = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const int d = KU * (t + 4 * (w / (KU / 4))) + 4 * (w % (KU / 4));
        raw[w] = h < heads ? *reinterpret_cast<const uint2*>(qp + d) : make_uint2(0, 0);
        const float2 x = unpack2<T>(raw[w].x), y = unpack2<T>(raw[w].y);
        most = fmaxf(fmaxf(most, fmaxf(kv8_magnitude(x.x), kv8_magnitude(x.y))), fmaxf(kv8_magnitude(y.x), kv8_magnitude(y.y)));
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int e = min(120, max(-100, (int)(__float_as_uint(most) >> 23) - 127));
      const float inv = kv8_pow2(-e);
      cq[n] = a.scale * 1.4426950408889634f * kv8_pow2(e);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const float2 x = unpack2<T>(raw[w].x), y = unpack2<T>(raw[w].y);
        qa[w][2 * n] = pack_f16(x.x * inv, x.y * inv);
        qa[w][2 * n + 1] = pack_f16(y.x * inv, y.y * inv);
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

    auto compute = [&](int step, const uint32_t* k, uint32_t* v, float kscale, float vscale) {
      float sc[2][4];  // scores of the tokens 0-7 and 8-15: [head g: 2t, 2t + 1][head g + 8: 2t, 2t + 1]
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[r][i] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const uint32_t b0 = kv8_decode2(k[r * KW + w]), b1 = kv8_decode2_hi(k[r * KW + w]);
          mma_f16(sc[r], qa[w][0], NT == 2 ? qa[w][2 * (NT - 1)] : 0u, qa[w][1], NT == 2 ? qa[w][2 * (NT - 1) + 1] : 0u, b0, b1);
        }
      }
      const int tok = (base + step) * KA_STEP;
      const bool edge = tok < tok_lo || tok + KA_STEP > tok_hi || vscale == 0.f;
      if (edge) {  // tokens out of sight: what stands there may be anything, NaN included
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int x = tok + (r >> 1) * 8 + 2 * t + (r & 1);
          if (x < tok_lo || x >= tok_hi || vscale == 0.f) {
            sc[r >> 1][r & 1] = -INFINITY;
            sc[r >> 1][2 + (r & 1)] = -INFINITY;
#pragma unroll
            for (int i = 0; i < VW; ++i) v[r * VW + i] = 0;
          }
        }
      }
      const float lv = vscale == 0.f ? 0.f : log2f(vscale), inv_v = vscale == 0.f ? 0.f : 1.f / vscale;
      uint32_t p[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float c = cq[n] * kscale;
        float x[4] = {fmaf(sc[0][2 * n], c, lv), fmaf(sc[0][2 * n + 1], c, lv), fmaf(sc[1][2 * n], c, lv), fmaf(sc[1][2 * n + 1], c, lv)};
        if (edge) {  // c may be 0 or negative: -inf again
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int y = tok + (r >> 1) * 8 + 2 * t + (r & 1);
            if (y < tok_lo || y >= tok_hi || vscale == 0.f) x[r] = -INFINITY;
          }
        }
        const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        if (__any_sync(0xffffffffu, top > m[n] + 8.f)) {
          float mx = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          mx = fmaxf(m[n], fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)));
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
    };

    // two steps a turn, so that the buffers' indexes are constants
    for (; s < s1; s += 2 * KA_WARPS) {
      const int sa = s + KA_WARPS, sb = s + 2 * KA_WARPS;
      if (sa < s1) {
        const int blk = blk_next;
        if (sb < s1) blk_next = page_of(sb);
        load(sa, blk, kw[1], vw[1], ks[1], vs[1]);
      }
      compute(s, kw[0], vw[0], ks[0], vs[0]);
      if (sa >= s1) break;
      if (sb < s1) {
        const int blk = blk_next;
        if (sb + KA_WARPS < s1) blk_next = page_of(sb + KA_WARPS);
        load(sb, blk, kw[0], vw[0], ks[0], vs[0]);
      }
      compute(sa, kw[1], vw[1], ks[1], vs[1]);
    }

    // join the warps
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
      if (t == 0) {
        sh_m[wid * HT + 8 * n + g] = m[n];
        sh_l[wid * HT + 8 * n + g] = l[n];
      }
#pragma unroll
      for (int i = 0; i < VW; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int d = VU * (g + 8 * (i / (VU / 4))) + 4 * (i % (VU / 4)) + 2 * half;  // and d + 1
          float* dst = sh_o + ((size_t)(wid * HT) + 8 * n + 2 * t) * D + d;
          *reinterpret_cast<float2*>(dst) = make_float2(o[2 * i + half][n][0], o[2 * i + half][n][2]);
          *reinterpret_cast<float2*>(dst + D) = make_float2(o[2 * i + half][n][1], o[2 * i + half][n][3]);
        }
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    float* part = a.part + ((size_t)2 * blockIdx.x + (u - s0 < first ? 0 : 1)) * HT * (D + 2);
    for (int i = tid; i < HT * D; i += KA_THREADS) {
      const int h = i / D, d = i % D;
      if (h >= heads) break;
      float mx = sh_m[h];
#pragma unroll
      for (int w = 1; w < KA_WARPS; ++w) mx = fmaxf(mx, sh_m[w * HT + h]);
      float acc = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < KA_WARPS; ++w) {
        const float f = fast_exp2(sh_m[w * HT + h] - mx);
        acc = fmaf(sh_o[(size_t)(w * HT + h) * D + d], f, acc);
        den = fmaf(sh_l[w * HT + h], f, den);
      }
      if (whole) {
        store1(reinterpret_cast<T*>(a.out) + ((size_t)b * a.Hk * a.G + kvh * a.G + h0 + h) * D + d, den != 0.f ? acc / den : 0.f);
      } else {
        part[h * (D + 2) + d] = acc;
        if (d == 0) {
          part[h * (D + 2) + D] = mx;
          part[h * (D + 2) + D + 1] = den;
        }
      }
    }
    __syncthreads();
    u += s1 - s0;
  }
}

// Rows that several blocks share: their parts in the order of the blocks.  One block per (sequence, row of the list).
template <int D, int HT, typename T>
__global__ void __launch_bounds__(KA_THREADS)
kv8_attn_join_kernel(const __grid_constant__ Kv8AttnArgs a, int blocks) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, row = blockIdx.y, rows_per_seq = a.Hk * a.tiles;
  __shared__ int sums[2][KA_WARPS];
  int before = 0, all = 0, lo, hi;
  for (int i = threadIdx.x; i < a.B; i += KA_THREADS) {
    const int n = kv8_steps(a, i, lo, hi);
    all += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sums[0][threadIdx.x >> 5] = before;
    sums[1][threadIdx.x >> 5] = all;
  }
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < KA_WARPS; ++w) {
    before += sums[0][w];
    all += sums[1][w];
  }
  const int steps = kv8_steps(a, b, lo, hi);
  if (steps == 0) return;
  const long long run = kv8_run(a, (long long)all * rows_per_seq, blocks);
  const long long u0 = (long long)before * rows_per_seq + (long long)row * steps, u1 = u0 + steps;
  const long long c0 = u0 / run, c1 = (u1 - 1) / run;
  if (c0 == c1) return;  // one block had all of it
  const int kvh = row / a.tiles, h0 = (row % a.tiles) * HT, heads = min(HT, a.G - h0);
  for (int i = threadIdx.x; i < heads * D; i += KA_THREADS) {
    const int h = i / D, d = i % D;
    float mx = KA_NONE, acc = 0.f, den = 0.f;
    for (long long c = c0; c <= c1; ++c) {
      const float* p = a.part + ((size_t)2 * c + (u0 < c * run ? 0 : 1)) * HT * (D + 2) + h * (D + 2);
      const float pm = p[D], up = fmaxf(mx, pm), fa = fast_exp2(mx - up), fb = fast_exp2(pm - up);
      acc = fmaf(p[d], fb, acc * fa);
      den = fmaf(p[D + 1], fb, den * fa);
      mx = up;
    }
    store1(reinterpret_cast<T*>(a.out) + ((size_t)b * a.Hk * a.G + kvh * a.G + h0 + h) * D + d, den != 0.f ? acc / den : 0.f);
  }
}

inline int kv8_head_tile(int D, int G) { return G <= 8 || D > 128 ? 8 : 16; }
inline int kv8_attn_blocks(int D, int HT) { return trlb_host::sm_count() * kv8_attn_per_sm(D, HT); }

template <int D, int HT, typename T>
int kv8_attn_launch(Kv8AttnArgs& a, cudaStream_t st) {
  const size_t smem = (size_t)KA_WARPS * HT * (D + 2) * 4 + (size_t)(a.B + 1) * 4;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kv8_attn_kernel<D, HT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 72 * 1024);
    if (e != cudaSuccess) return (int)e;
  }
  const int blocks = kv8_attn_blocks(D, HT);
  const bool pdl = trlb_host::pdl_enabled();
  cudaError_t e = trlb_host::launch_kernel(kv8_attn_kernel<D, HT, T>, dim3(blocks), dim3(KA_THREADS), smem, st, pdl, a);
  if (e != cudaSuccess) return (int)e;
  return (int)trlb_host::launch_kernel(kv8_attn_join_kernel<D, HT, T>, dim3(a.B, a.Hk * a.tiles), dim3(KA_THREADS), 0, st, pdl, a, blocks);
}
template <typename T>
int kv8_attn_pick(Kv8AttnArgs& a, int D, cudaStream_t st) {
  const int ht = kv8_head_tile(D, a.G);
  a.tiles = (a.G + ht - 1) / ht;
  if (a.Hk * a.tiles > 65535) return -5;
  switch (D) {
    case 64: return ht == 8 ? kv8_attn_launch<64, 8, T>(a, st) : kv8_attn_launch<64, 16, T>(a, st);
    case 96: return ht == 8 ? kv8_attn_launch<96, 8, T>(a, st) : kv8_attn_launch<96, 16, T>(a, st);
    case 128: return ht == 8 ? kv8_attn_launch<128, 8, T>(a, st) : kv8_attn_launch<128, 16, T>(a, st);
    case 256: return kv8_attn_launch<256, 8, T>(a, st);
  }
  return -1;
}

}  // namespace trlb

using namespace trlb;

// fp32 words of scratch that a call needs: parts of rows that several blocks share
TRLB_API long long trlb_kv8_attn_scratch(int Hq, int Hk, int D) {
  const int ht = kv8_head_tile(D, Hq / Hk);
  return 2ll * kv8_attn_blocks(D, ht) * ht * (D + 2);
}

// q [B, Hq, D] bf16 (dtype 0) or fp16 (1) with strides in elements (multiples of 4, rows 8 bytes aligned); out dense.
// page_size a power of two, 16 or more.  window 0: everything.  Rows with seq_len < 0 get zeros.
TRLB_API int trlb_kv8_decode_attn(const void* q, int dtype, long long q_row, long long q_head, const void* k_codes,
                                  const void* v_codes, const float* k_scale, const float* v_scale, int pages, int page_size,
                                  const int* table, int table_rows, int max_blocks, const int* seq_lens, const int* slots,
                                  int B, int Hq, int Hk, int D, float scale, int window, float* part, void* out, int* status,
                                  cudaStream_t st) {
  if (B == 0) return 0;
  if (Hk <= 0 || Hq <= 0 || Hq % Hk || B > KA_MAX_SEQS || window < 0) return -2;
  if (page_size < KA_STEP || (page_size & (page_size - 1))) return -3;
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  Kv8AttnArgs a{q, q_row, q_head, (const uint8_t*)k_codes, (const uint8_t*)v_codes, k_scale, v_scale, table, seq_lens, slots,
                out, part, status, pages, Hk, Hq / Hk, 1, shift, table_rows, max_blocks, B, window, KA_WARPS, scale};
  if (dtype == 0) return kv8_attn_pick<__nv_bfloat16>(a, D, st);
  if (dtype == 1) return kv8_attn_pick<__half>(a, D, st);
  return -4;
}
