// Keys and values of new tokens into the 8-bit paged cache.
//
//   kv8_append_pages   packed pieces of any length (prompts, pieces that continue a sequence): one block per page and head
//   kv8_append_rows    one token per sequence: one warp per row and head
//   kv8_rope_append    the same behind RoPE (and the norms of q and k), fed by the QKV product of a decode step
//
// Cache: codes [pages, heads, page size, head dim] e4m3 and scales [pages, heads] fp32, for keys and for values.  With a the
// largest magnitude of the new tokens in a page, the page's scale becomes 2^e(a) where its first row is among them and
// max(scale, 2^e(a)) otherwise; in the second case the rows that stand before are brought to the new scale.  Rows behind
// the last token are left as they are.
#include <cuda_fp16.h>
#include <type_traits>

#include "kv8.cuh"

namespace trlb {

enum { SITE_KV8_APPEND = 1400, SITE_KV8_ROWS = 1401, SITE_KV8_ROPE = 1402 };

// One of two parameters: an index that is not known when compiled would copy them to local memory first (84 us instead of 70 for
// 134 million bf16 values).
template <typename P>
__device__ __forceinline__ P of_side(const P (&two)[2], int which) { return which ? two[1] : two[0]; }

struct Kv8Cache {
  uint8_t* codes[2];  // keys, values
  float* scale[2];
  int pages, heads, page_size, dim;
};

// Where position `pos` of sequence row `slot` lives, or -1 (reported) where the table has no such page.
__device__ __forceinline__ int kv8_page_of(const int* table, int rows, int max_blocks, int slot, int index, int pages,
                                           int* status, int site) {
  if (slot < 0 || slot >= rows || index >= max_blocks) {
    report_error(status, ERR_BOUNDS, site, slot);
    return -1;
  }
  const int blk = table[(size_t)slot * max_blocks + index];
  if (blk < 0 || blk >= pages) {
    report_error(status, ERR_BOUNDS, site, blk);
    return -1;
  }
  return blk;
}

__device__ __forceinline__ uint32_t kv8_again4(uint32_t c, float ratio) {
  const uint32_t lo = kv8_decode2(c), hi = kv8_decode2_hi(c);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return kv8_encode2(a.x, a.y, ratio) | (kv8_encode2(b.x, b.y, ratio) << 16);
}
// Rows before the new ones: codes * old scale / new scale, rounded again.  `bytes` is a multiple of 16.
__device__ __forceinline__ void kv8_again(uint8_t* codes, int bytes, float ratio, int tid, int threads) {
  uint4* p = reinterpret_cast<uint4*>(codes);
  for (int i = tid; i < bytes / 16; i += threads) {
    uint4 u = p[i];
    u.x = kv8_again4(u.x, ratio);
    u.y = kv8_again4(u.y, ratio);
    u.z = kv8_again4(u.z, ratio);
    u.w = kv8_again4(u.w, ratio);
    p[i] = u;
  }
}

// Eight values as they stand in memory, and as floats.
template <typename T>
struct Raw8 { uint4 u[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ void load8(const T* p, Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
}
__device__ __forceinline__ void floats8(const Raw8<__nv_bfloat16>& r, float (&x)[8]) {
  const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack_bf16(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void floats8(const Raw8<__half>& r, float (&x)[8]) {
  const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void floats8(const Raw8<float>& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[4 * i] = __uint_as_float(r.u[i].x);
    x[4 * i + 1] = __uint_as_float(r.u[i].y);
    x[4 * i + 2] = __uint_as_float(r.u[i].z);
    x[4 * i + 3] = __uint_as_float(r.u[i].w);
  }
}
// Largest magnitude of some values as the type's bits (ordered like the magnitudes; infinities and NaN are at least `special`).
template <typename T>
struct Bits;
template <>
struct Bits<__nv_bfloat16> {
  static constexpr uint32_t special = 0x7f80u;
  static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b << 16); }
};
template <>
struct Bits<__half> {
  static constexpr uint32_t special = 0x7c00u;
  static __device__ __forceinline__ float value(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }
};
template <>
struct Bits<float> {
  static constexpr uint32_t special = 0x7f800000u;
  static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b); }
};
template <typename T>
__device__ __forceinline__ uint32_t largest8(const Raw8<T>& r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
    const uint32_t w[4] = {r.u[i].x, r.u[i].y, r.u[i].z, r.u[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) m = sizeof(T) == 2 ? __vmaxu2(m, w[j] & 0x7fff7fffu) : max(m, w[j] & 0x7fffffffu);
  }
  return sizeof(T) == 2 ? max(m & 0xffffu, m >> 16) : m;
}
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }

template <typename T>
struct Kv8Source {
  const T* x[2];               // keys, values: [tokens, heads, dim], the last dimension dense
  long long tok[2], head[2];   // strides in elements
};

// The new rows of pages, read once into registers: their largest magnitude decides the scale, then they are written.  A group
// of threads (a warp for pages of up to 2048 values, else the block) takes one page and ITEMS of its 2 x heads tiles (head, keys
// or values), whose loads are all under way together.  Bound by the bytes, 2 or 4 read and 1 written a value: 65536 tokens of
// 8 heads and 128 dimensions in bf16 take 71 us, 5.7 TB/s; 16 prompts of up to 1024 tokens 7.8 us, a page's chain of reads.
template <typename T, int VECS, int ITEMS, bool WARP>
__global__ void __launch_bounds__(256, sizeof(T) == 4 || VECS == 16 ? 2 : 4)
kv8_append_pages_kernel(Kv8Source<T> src, Kv8Cache c, const int* __restrict__ table, int table_rows, int max_blocks,
                        const int* __restrict__ starts, const int* __restrict__ cu, const int* __restrict__ slots, int n,
                        int tokens, int pages_per_seq, int* status) {
  constexpr int GROUP = WARP ? 32 : 256, GROUPS = 256 / GROUP;
  const int in = threadIdx.x % GROUP, wid = threadIdx.x >> 5;
  const long long item = (long long)blockIdx.x * GROUPS + threadIdx.x / GROUP;
  __shared__ uint32_t part[ITEMS][8];
  const int seq = (int)(item / pages_per_seq), nth = (int)(item % pages_per_seq);
  if (seq >= n) return;  // whole groups leave, here and below
  const int start = starts[seq];
  const int t0 = cu[seq], t1 = min(cu[seq + 1], tokens);
  if (start < 0 || t0 < 0 || t1 <= t0) return;
  const int bs = c.page_size, D = c.dim;
  const int index = start / bs + nth;                   // page of the sequence
  const int p0 = max(start, index * bs);                // positions of its new rows
  const long long end = (long long)start + (t1 - t0);
  const int p1 = (int)min(end, (long long)(index + 1) * bs);
  if (p1 <= p0) return;
  const int blk = kv8_page_of(table, table_rows, max_blocks, slots ? slots[seq] : seq, index, c.pages, status, SITE_KV8_APPEND);
  if (blk < 0) return;
  const int row0 = p0 - index * bs, vecs = D / 8, count = (p1 - p0) * vecs, first = blockIdx.y * ITEMS;
  auto side = [](int tile, int k) { return ITEMS % 2 == 0 ? k & 1 : tile & 1; };  // keys or values: known when compiled
  Raw8<T> raw[ITEMS][VECS];
  uint32_t top[ITEMS];
  float old[ITEMS];
  if (GROUP % vecs == 0) {  // a thread's vectors stand below each other: all but head dim 96
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int tile = first + k, which = side(tile, k);
      const T* x = of_side(src.x, which) + (long long)(t0 + (p0 - start) + in / vecs) * of_side(src.tok, which) + (long long)(tile >> 1) * of_side(src.head, which) + in % vecs * 8;
      const long long step = GROUP / vecs * of_side(src.tok, which);
      if (tile < 2 * c.heads)
#pragma unroll
        for (int j = 0; j < VECS; ++j)
          if (in + j * GROUP < count) load8<T>(x + j * step, raw[k][j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      const int i = in + j * GROUP;
      const long long row = t0 + (p0 - start) + i / vecs;
      const int col = (i % vecs) * 8;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
        const int tile = first + k, which = side(tile, k);
        if (i < count && tile < 2 * c.heads)
          load8<T>(of_side(src.x, which) + row * of_side(src.tok, which) + (long long)(tile >> 1) * of_side(src.head, which) + col, raw[k][j]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int tile = first + k;
    old[k] = row0 > 0 && tile < 2 * c.heads ? of_side(c.scale, side(tile, k))[(size_t)blk * c.heads + (tile >> 1)] : 0.f;
    top[k] = 0;
#pragma unroll
    for (int j = 0; j < VECS; ++j)
      if (in + j * GROUP < count && tile < 2 * c.heads) top[k] = max(top[k], largest8<T>(raw[k][j]));
    top[k] = __reduce_max_sync(0xffffffffu, top[k]);
    if (!WARP && (threadIdx.x & 31) == 0) part[k][wid] = top[k];
  }
  if (!WARP) __syncthreads();
  else __syncwarp();  // every lane has read the old scales
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int tile = first + k, which = side(tile, k);
    if (tile >= 2 * c.heads) break;
    if (!WARP)
#pragma unroll
      for (int w = 0; w < 8; ++w) top[k] = max(top[k], part[k][w]);
    float amax = Bits<T>::value(top[k]);
    const bool special = top[k] >= Bits<T>::special;  // an infinity or NaN among them: rare, so the scale is found again without
    if (special) {
      amax = 0.f;
#pragma unroll
      for (int j = 0; j < VECS; ++j) {
        float v[8];
        floats8(raw[k][j], v);
        if (in + j * GROUP < count)
#pragma unroll
          for (int e = 0; e < 8; ++e) amax = fmaxf(amax, kv8_magnitude(v[e]));
      }
      amax = warp_max(amax);
      if (!WARP) {
        __shared__ float again[8];
        __syncthreads();
        if ((threadIdx.x & 31) == 0) again[wid] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) amax = fmaxf(amax, again[w]);
      }
    }
    const size_t at = (size_t)blk * c.heads + (tile >> 1);
    uint8_t* page = of_side(c.codes, which) + at * bs * D;
    const float now = fmaxf(old[k], kv8_pow2(kv8_exponent(amax)));
    if (row0 > 0 && now > old[k]) kv8_again(page, row0 * D, old[k] / now, in, GROUP);
    const float inv = 1.f / now;
#pragma unroll
    for (int j = 0; j < VECS; ++j) {
      const int i = in + j * GROUP;
      if (i < count) {
        float v[8];
        floats8(raw[k][j], v);
        uint2 u;
        if (special) {
          u.x = kv8_encode2(v[0], v[1], inv) | (kv8_encode2(v[2], v[3], inv) << 16);
          u.y = kv8_encode2(v[4], v[5], inv) | (kv8_encode2(v[6], v[7], inv) << 16);
        } else {
          u.x = kv8_encode2_finite(v[0], v[1], inv) | (kv8_encode2_finite(v[2], v[3], inv) << 16);
          u.y = kv8_encode2_finite(v[4], v[5], inv) | (kv8_encode2_finite(v[6], v[7], inv) << 16);
        }
        reinterpret_cast<uint2*>(page + row0 * D)[i] = u;
      }
    }
    if (in == 0) of_side(c.scale, which)[at] = now;
  }
}

// One warp per (sequence, head, keys or values): the row of one token.
template <typename T>
__global__ void __launch_bounds__(128)
kv8_append_rows_kernel(Kv8Source<T> src, Kv8Cache c, const int* __restrict__ table, int table_rows, int max_blocks,
                       const int* __restrict__ starts, const int* __restrict__ slots, int n, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (item >= (long long)n * c.heads * 2) return;
  const int which = (int)(item & 1), head = (int)((item >> 1) % c.heads), seq = (int)((item >> 1) / c.heads);
  const int pos = starts[seq];
  if (pos < 0) return;
  const int bs = c.page_size, D = c.dim, row = pos % bs;
  const int blk = kv8_page_of(table, table_rows, max_blocks, slots ? slots[seq] : seq, pos / bs, c.pages, status, SITE_KV8_ROWS);
  if (blk < 0) return;
  const T* x = of_side(src.x, which) + (long long)seq * of_side(src.tok, which) + (long long)head * of_side(src.head, which);
  float v[8], amax = 0.f;  // D <= 256
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    v[i] = d < D ? as_float(x[d]) : 0.f;
    amax = fmaxf(amax, kv8_magnitude(v[i]));
  }
  uint8_t* page = of_side(c.codes, which) + ((size_t)blk * c.heads + head) * bs * D;
  float* scale = of_side(c.scale, which) + (size_t)blk * c.heads + head;
  const float old = row > 0 ? *scale : 0.f;
  const float now = fmaxf(old, kv8_pow2(kv8_exponent(warp_max(amax))));
  if (row > 0 && now > old) kv8_again(page, row * D, old / now, lane, 32);
  const float inv = 1.f / now;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (d < D) page[row * D + d] = (uint8_t)kv8_encode2(v[i], 0.f, inv);
  }
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *scale = now;
}

// The decode step's QKV row -> rotated queries and a row of the cache.  F32: the row arrives as fp32 sums of the stream-K
// product, is cleared here, and gets bias and norms; else it is a finished bf16 row.  Values are rounded to bf16 where the
// bf16 cache's kernels round them (after the bias, after the norm, after the rotation), so the two caches differ by their
// last rounding only.  One warp per (token, head); a lane owns the rotation pairs (f, f + dim / 2), f = lane, lane + 32.  Bound by
// one chain: length, sums, table entry, scale, the page's earlier rows where the scale grows.  64 tokens of 28 and 4 heads of 128
// take 3.5 us (their bytes 0.44), into the 16-bit cache 3.9; 256 tokens of 32 and 8 heads 14.4 us (2.3), 15.8.
template <bool F32>
__global__ void __launch_bounds__(256)
kv8_rope_append_kernel(void* __restrict__ qkv, long long row_stride, const __nv_bfloat16* __restrict__ bias,
                       const __nv_bfloat16* __restrict__ q_norm, const __nv_bfloat16* __restrict__ k_norm, float norm_eps,
                       const int* __restrict__ seq_lens, const int* __restrict__ slot_ids, const int* __restrict__ table,
                       int table_rows, int max_blocks, __nv_bfloat16* __restrict__ q_out, Kv8Cache c, int B, int Hq,
                       float log2_theta, const int* __restrict__ pos_delta, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int D = c.dim, half = D >> 1, heads = Hq + 2 * c.heads;
  const int lane = threadIdx.x & 31;
  const int item = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (item >= B * heads) return;
  const int b = item / heads, head = item % heads;
  const int slot = slot_ids ? slot_ids[b] : b;
  const bool known = slot >= 0 && slot < table_rows;  // a slot that the table does not have: reported, and treated as idle
  if (!known && lane == 0) report_error(status, ERR_BOUNDS, SITE_KV8_ROPE, slot);
  const int pos = known ? seq_lens[slot] : -1;
  const size_t base = (size_t)b * row_stride + (size_t)head * D;
  float lo[2], hi[2], ss = 0.f;
  auto bf = [](float x) { return __bfloat162float(__float2bfloat16(x)); };
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int f = lane + 32 * j;
    lo[j] = hi[j] = 0.f;
    if (f >= half) continue;
    if constexpr (F32) {
      float* src = reinterpret_cast<float*>(qkv) + base;
      lo[j] = src[f];
      hi[j] = src[half + f];
      src[f] = 0.f;
      src[half + f] = 0.f;
      if (bias) {
        lo[j] += __bfloat162float(bias[(size_t)head * D + f]);
        hi[j] += __bfloat162float(bias[(size_t)head * D + half + f]);
      }
      lo[j] = bf(lo[j]);
      hi[j] = bf(hi[j]);
    } else {
      const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(qkv) + base;
      lo[j] = __bfloat162float(src[f]);
      hi[j] = __bfloat162float(src[half + f]);
    }
    ss += lo[j] * lo[j] + hi[j] * hi[j];
  }
  if (pos < 0) return;  // idle slot: sums are dropped
  const __nv_bfloat16* nw = head < Hq ? q_norm : (head < Hq + c.heads ? k_norm : nullptr);
  if (nw != nullptr) {
    const float rstd = rsqrtf(warp_sum(ss) / (float)D + norm_eps);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int f = lane + 32 * j;
      if (f < half) {
        lo[j] = bf(lo[j] * rstd * __bfloat162float(nw[f]));
        hi[j] = bf(hi[j] * rstd * __bfloat162float(nw[half + f]));
      }
    }
  }
  const bool value = head >= Hq + c.heads;
  if (!value) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int f = lane + 32 * j;
      if (f >= half) continue;
      const float inv = exp2f(-log2_theta * (float)(2 * f) / (float)D);
      float sn, cs;
      sincosf((float)(pos + (pos_delta ? pos_delta[slot] : 0)) * inv, &sn, &cs);
      const float l = lo[j], h = hi[j];
      lo[j] = bf(l * cs - h * sn);
      hi[j] = bf(h * cs + l * sn);
    }
  }
  if (head < Hq) {
    __nv_bfloat16* dst = q_out + ((size_t)b * Hq + head) * D;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int f = lane + 32 * j;
      if (f < half) {
        dst[f] = __float2bfloat16(lo[j]);
        dst[half + f] = __float2bfloat16(hi[j]);
      }
    }
    return;
  }
  const int which = value ? 1 : 0, kh = head - Hq - which * c.heads, bs = c.page_size, row = pos % bs;
  const int blk = kv8_page_of(table, table_rows, max_blocks, slot, pos / bs, c.pages, status, SITE_KV8_ROPE);
  if (blk < 0) return;
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j) amax = fmaxf(amax, fmaxf(kv8_magnitude(lo[j]), kv8_magnitude(hi[j])));
  uint8_t* page = of_side(c.codes, which) + ((size_t)blk * c.heads + kh) * bs * D;
  float* scale = of_side(c.scale, which) + (size_t)blk * c.heads + kh;
  const float old = row > 0 ? *scale : 0.f;
  const float now = fmaxf(old, kv8_pow2(kv8_exponent(warp_max(amax))));
  if (row > 0 && now > old) kv8_again(page, row * D, old / now, lane, 32);
  const float inv = 1.f / now;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int f = lane + 32 * j;
    if (f < half) {
      const uint32_t u = kv8_encode2(lo[j], hi[j], inv);
      page[row * D + f] = (uint8_t)u;
      page[row * D + half + f] = (uint8_t)(u >> 8);
    }
  }
  __syncwarp();
  if (lane == 0) *scale = now;
}

template <typename T>
int kv8_append_launch(const Kv8Source<T>& src, const Kv8Cache& c, const int* table, int table_rows, int max_blocks,
                      const int* starts, const int* cu, const int* slots, int n, int tokens, int max_new, int* status,
                      cudaStream_t st) {
  if (cu == nullptr) {
    const long long warps = (long long)n * c.heads * 2;
    return (int)trlb_host::launch_kernel(kv8_append_rows_kernel<T>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, st,
                                         trlb_host::pdl_enabled(), src, c, table, table_rows, max_blocks, starts, slots, n,
                                         status);
  }
  const long long per = (max_new - 1) / c.page_size + 2;  // a piece may begin inside a page
  if (per * n > 2147483647ll) return -3;
  auto go = [&](auto vecs, auto items, auto warp) {
    constexpr int V = decltype(vecs)::value, I = decltype(items)::value;
    constexpr bool W = decltype(warp)::value;
    const unsigned groups = W ? 8 : 1;
    kv8_append_pages_kernel<T, V, I, W><<<dim3((unsigned)((per * n + groups - 1) / groups), (2 * c.heads + I - 1) / I), 256, 0, st>>>(
        src, c, table, table_rows, max_blocks, starts, cu, slots, n, tokens, (int)per, status);
    return (int)cudaGetLastError();
  };
  // 8 vectors of 16 bytes a thread, where a tile allows it: two tiles of 64 rows of 128 bf16 values, say
  using std::integral_constant;
  const int values = c.page_size * c.dim;
  if (values <= 1024) return go(integral_constant<int, 4>(), integral_constant<int, 2>(), std::true_type());
  if (values <= 2048) return go(integral_constant<int, 8>(), integral_constant<int, 1>(), std::true_type());
  if (values <= 4096) return go(integral_constant<int, 2>(), integral_constant<int, 4>(), std::false_type());
  if (values <= 8192) return go(integral_constant<int, 4>(), integral_constant<int, 2>(), std::false_type());
  if (values <= 16384) return go(integral_constant<int, 8>(), integral_constant<int, 1>(), std::false_type());
  if (values <= 32768) return go(integral_constant<int, 16>(), integral_constant<int, 1>(), std::false_type());
  return -6;
}

}  // namespace trlb

using namespace trlb;

// dtype: 0 bf16, 1 fp16, 2 fp32.  Rows of dim dense elements on 16 bytes.  cu null: one token per sequence (tokens == n).
struct Kv8AppendCall {
  const void *k, *v;
  void *k_codes, *v_codes;
  float *k_scale, *v_scale;
  const int *table, *starts, *cu, *slots;
  int* status;
  cudaStream_t stream;
  long long k_tok, k_head, v_tok, v_head;  // strides in elements
  int dtype, pages, heads, page_size, dim, table_rows, max_blocks, n, tokens, max_new;
};
TRLB_API int trlb_kv8_append(const Kv8AppendCall* call) {
  const Kv8AppendCall a = *call;
  if (a.n == 0 || a.tokens == 0) return 0;
  if (a.dim <= 0 || a.dim > 256 || a.dim % 16 || a.heads <= 0 || a.heads > 65535 || a.page_size <= 0) return -1;
  if (a.max_new < 1 || (a.cu == nullptr && a.tokens != a.n)) return -2;
  Kv8Cache c{{(uint8_t*)a.k_codes, (uint8_t*)a.v_codes}, {a.k_scale, a.v_scale}, a.pages, a.heads, a.page_size, a.dim};
  auto go = [&](auto* type) {
    using T = std::remove_pointer_t<decltype(type)>;
    const Kv8Source<T> src{{(const T*)a.k, (const T*)a.v}, {a.k_tok, a.v_tok}, {a.k_head, a.v_head}};
    return kv8_append_launch(src, c, a.table, a.table_rows, a.max_blocks, a.starts, a.cu, a.slots, a.n, a.tokens, a.max_new,
                             a.status, a.stream);
  };
  if (a.dtype == 0) return go((__nv_bfloat16*)nullptr);
  if (a.dtype == 1) return go((__half*)nullptr);
  if (a.dtype == 2) return go((float*)nullptr);
  return -4;
}

// qkv: bf16 rows (f32 == 0) or fp32 sums that are cleared.  bias / norms / pos_delta / slot_ids may be null.  dim <= 128.
// seq_lens and pos_delta have an entry for each slot that is used, with slot_ids for each row of the table.
TRLB_API int trlb_kv8_rope_append(void* qkv, int f32, long long row_stride, const void* bias, const void* q_norm,
                                  const void* k_norm, float norm_eps, const int* seq_lens, const int* slot_ids,
                                  const int* table, int table_rows, int max_blocks, void* q_out, void* k_codes, void* v_codes,
                                  float* k_scale, float* v_scale, int pages, int heads, int page_size, int dim, int B, int Hq,
                                  float theta, const int* pos_delta, int* status, cudaStream_t st) {
  if (B == 0) return 0;
  if (dim <= 0 || dim > 128 || dim % 16 || heads <= 0 || page_size <= 0) return -1;
  const long long items = (long long)B * (Hq + 2 * heads);
  if (items > 67108863ll) return -3;
  Kv8Cache c{{(uint8_t*)k_codes, (uint8_t*)v_codes}, {k_scale, v_scale}, pages, heads, page_size, dim};
  const dim3 grid((unsigned)((items + 7) / 8));
  if (f32)
    return (int)trlb_host::launch_kernel(kv8_rope_append_kernel<true>, grid, dim3(256), 0, st, trlb_host::pdl_enabled(), qkv,
                                         row_stride, (const __nv_bfloat16*)bias, (const __nv_bfloat16*)q_norm,
                                         (const __nv_bfloat16*)k_norm, norm_eps, seq_lens, slot_ids, table, table_rows,
                                         max_blocks, (__nv_bfloat16*)q_out, c, B, Hq, log2f(theta), pos_delta, status);
  return (int)trlb_host::launch_kernel(kv8_rope_append_kernel<false>, grid, dim3(256), 0, st, trlb_host::pdl_enabled(), qkv,
                                       row_stride, (const __nv_bfloat16*)nullptr, (const __nv_bfloat16*)q_norm,
                                       (const __nv_bfloat16*)k_norm, norm_eps, seq_lens, slot_ids, table, table_rows,
                                       max_blocks, (__nv_bfloat16*)q_out, c, B, Hq, log2f(theta), pos_delta, status);
}
