// Sampling with temperature, top-k, top-p and min-p from one random word per row.
//
//   z = logit / max(temperature, 1e-6) in fp32; NaN counts as -inf, what is above fp32's largest number as that number
//   top-k keeps what is at least the k-th largest z (equals of the k-th too); 0 keeps all
//   top-p keeps, most likely first and the lower column first among equals, each token before which at most
//         top_p of the mass of what top-k kept stands
//   min-p keeps z >= max z + log(min_p)
//   token = argmax over what is kept of z - log(-log u), u = (hash(word of the row, column) + 1/2) / 2^32; of z where
//   temperature is 0; its log-probability is that in the distribution over what is kept
//
// All filters are one border: the last token kept, in the order "larger z, then lower column".  A row is read by the blocks
// of a cluster.  What bounds it is the work per logit (the row's bytes stay in the second-level cache after the first pass) and
// the latency of the few exchanges between the blocks; so logits are divided only where z decides, and the border is found in as
// few passes as the row allows.  Logits of 16 bits have the order of their z.  Neighbouring fp32 logits can have one z, whichever
// way round they stand: their lists hold z, and the numbers that they are compared with are the smallest logits of a z (least_of).
//   1. the maximum and the mass, each thread with a running maximum of its own;
//   2. candidates for the kept tokens: with top-k of C blocks what is not below the k/C-th largest of the threads' maxima of any
//      (k logits are at least that large), with top-p alone what is not lighter than (1 - top_p) mass / V (lighter ones together
//      are less than what top-p leaves out).  Where one block's list holds them, it finds the border there and draws: done.
//   3. otherwise a histogram of the distances to the maximum.  From counts alone the bins bound the mass above each of them from
//      both sides, which brackets the border; the tokens of the bracket are listed, and the exact mass above it says which of
//      them is the last.  A bracket with too many tokens for the list is cut again by histograms over the logits' bits.
//   4. a last pass over the row draws among what is kept.
// A row that fits into the shared memory of a cluster is read once and stays there for all of it, larger ones are read again for
// each pass (SfSampler::fast); the few rows that need what fast() leaves out are read again and, where their order is not that of
// z, divided in each pass (SfSampler::run).
// Measured: one row of 152064 bf16 logits with top-k 20 and top-p 0.8 13.8 us; 64 rows with top-p 0.95 64 us (32 rows 48 us), of which the
// flattest row's 60 us are: load and mass 8, list given up 3, histogram 9, its border's bins 8, draw 19, list of the bracket 4,
// border 5, last draw 3; 256 rows of 128256 fp32 logits with parameters of all kinds 114 us.  run(), which top-k above 512 (256 for
// each block of the cluster) needs: 64 rows of 152064 bf16 logits 48 us at top-k 600, 51 at 1000, 107 at 2000, with top-k 500 29 us; fp32
// logits at temperature 0.7, which it divides in each pass, 53, 55 and 105 us, at temperature 1 44, 46 and 89.
// Counts and the sums over lists are integers, other sums are taken in a fixed order: results do not depend on timing.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cstddef>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace trlb {

constexpr int SF_THREADS = 512, SF_WARPS = SF_THREADS / 32;  // two blocks an SM
constexpr int SF_EACH = 4;         // bins of a thread: SF_BINS / SF_THREADS
constexpr int SF_BINS = 2048;      // histogram bins; the last one holds all that lies further below
constexpr int SF_LIST = 2048;      // tokens that the list holds
constexpr int SF_CUT = 1024;       // and the cut around the border; more are sorted in the list itself
constexpr int SF_FEW = 64;          // of so few tokens each is compared with all others
constexpr int SF_HELD = 5120;      // 16-byte vectors of a row in a block's shared memory, at most: with it two blocks an SM
constexpr float SF_FINE = 1024.f;  // parts of a bin in which the histogram adds up where in the bin its tokens lie
// Temperatures from here on: below, few tokens have a weight, and rounding z shows in it.  Up to SF_HIGH z is no denormal number where
// that would make one z of two 16-bit logits.
constexpr float SF_LOW = 0.015625f, SF_HIGH = 32768.f;
constexpr int SF_BATCH = 16;       // logits that a thread loads at once
constexpr float SF_MAX = 3.4028234663852886e38f;
constexpr float SF_LOG2E = 1.4426950408889634f;
constexpr double SF_UNIT = 17592186044416.;  // 2^44: weights in sums over lists are whole multiples of 1 / SF_UNIT

struct SampleArgs {
  const void* logits;
  long long row_stride;
  int V;
  const float *temperature, *top_p, *min_p;  // per row, or null: the values below
  const int* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  const uint32_t* words;  // per row, or null: of seed, step and row
  uint32_t seed;
  const int* step_ptr;
  int *tok;
  float* logp;
};

__device__ __forceinline__ uint32_t sf_hash(uint32_t x) {
  x ^= x >> 16; x *= 0x7feb352dU; x ^= x >> 15; x *= 0x846ca68bU; x ^= x >> 16;
  return x;
}
// The random bits of a column: u = (h + 1/2) / 2^32.
__device__ __forceinline__ uint32_t sf_bits(uint32_t word, uint32_t col) {
  return sf_hash(sf_hash(word ^ sf_hash(col * 0x85EBCA6BU + 0x165667B1U)) + col);
}
// -log(-log u): both halves of (0, 1) in the form that keeps their precision
__device__ __noinline__ float sf_gumbel(uint32_t h) {
  float e;
  if (h & 0x80000000u) e = -log1pf(-((float)(~h) + 0.5f) * 2.3283064365386963e-10f);
  else e = -logf(((float)h + 0.5f) * 2.3283064365386963e-10f);
  return -logf(e);
}
__device__ __forceinline__ float sf_quotient(float x, float t) { return fminf(__fdiv_rn(x, t), SF_MAX); }
// The same from the 24-bit numbers and fast logarithms of trlb_sample, so that one seed gives the same draws there and here.
// (The largest number rounds to 1, whose logarithm would let its token win whatever its logit: it counts as 1 - 2^-25.)
__device__ __forceinline__ float sf_gumbel_as_sampler(uint32_t h) {
  const float u = ((float)(h >> 8) + 0.5f) * (1.0f / 16777216.0f);
  return -__logf(fmaxf(-__logf(u), 2.98023224e-8f));
}
// Orders floats as unsigned integers.
__device__ __forceinline__ uint32_t sf_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sf_unkey(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ float sf_load(const float* p, long long i) { return p[i]; }
__device__ __forceinline__ float sf_load(const __nv_bfloat16* p, long long i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ float sf_load(const __half* p, long long i) { return __half2float(p[i]); }
template <typename T>
__device__ __forceinline__ void sf_unpack(uint4 u, float* x);
template <>
__device__ __forceinline__ void sf_unpack<float>(uint4 u, float* x) {
  x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
}
template <>
__device__ __forceinline__ void sf_unpack<__nv_bfloat16>(uint4 u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 f = unpack_bf16(w[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}
template <>
__device__ __forceinline__ void sf_unpack<__half>(uint4 u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x; x[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ T sf_lowest();
template <>
__device__ __forceinline__ float sf_lowest<float>() { return -INFINITY; }
template <>
__device__ __forceinline__ __nv_bfloat16 sf_lowest<__nv_bfloat16>() { return __ushort_as_bfloat16((unsigned short)0xff80); }
template <>
__device__ __forceinline__ __half sf_lowest<__half>() { return __ushort_as_half((unsigned short)0xfc00); }
// NaN -> -inf (a maximum drops it), nothing above cap, one zero of both.
__device__ __forceinline__ float sf_clean1(float y, float cap) { return fminf(fmaxf(y, -INFINITY), cap) + 0.f; }
template <typename T>
__device__ __forceinline__ void sf_clean(uint4& u);
template <>
__device__ __forceinline__ void sf_clean<float>(uint4& u) {
  u.x = __float_as_uint(sf_clean1(__uint_as_float(u.x), INFINITY));
  u.y = __float_as_uint(sf_clean1(__uint_as_float(u.y), INFINITY));
  u.z = __float_as_uint(sf_clean1(__uint_as_float(u.z), INFINITY));
  u.w = __float_as_uint(sf_clean1(__uint_as_float(u.w), INFINITY));
}
template <>
__device__ __forceinline__ void sf_clean<__nv_bfloat16>(uint4& u) {
  const __nv_bfloat162 lo = __bfloat162bfloat162(sf_lowest<__nv_bfloat16>()), zero = __bfloat162bfloat162(__float2bfloat16(0.f));
  __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __hadd2(__hmax2(p[i], lo), zero);
}
template <>
__device__ __forceinline__ void sf_clean<__half>(uint4& u) {
  const __half2 lo = __half2half2(sf_lowest<__half>()), zero = __half2half2(__float2half(0.f));
  __half2* p = reinterpret_cast<__half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __hadd2(__hmax2(p[i], lo), zero);
}

// Four of them over t.
__device__ __noinline__ float4 sf_over(float4 y, float t) {
  return make_float4(sf_clean1(__fdiv_rn(y.x, t), SF_MAX), sf_clean1(__fdiv_rn(y.y, t), SF_MAX), sf_clean1(__fdiv_rn(y.z, t), SF_MAX),
                     sf_clean1(__fdiv_rn(y.w, t), SF_MAX));
}

struct SfShared {
  unsigned hist[SF_BINS];
  union {
    unsigned where[SF_BINS];          // sums of the tokens' places in their bins
    unsigned cumul[SF_BINS];          // tokens up to and with a bin
    unsigned long long cut[SF_CUT];   // the part of the list around the border
  };
  unsigned long long list[SF_LIST];   // ~key << 32 | column: ascending is "larger logit, then lower column"
  double red[2][SF_WARPS];
  float warp_best[SF_WARPS], warp_z[SF_WARPS];
  int warp_col[SF_WARPS];
  unsigned long long sum[SF_WARPS];
  double mass, first_mass, sums[2];   // this block's shares of sums
  double kept;                        // mass down to the border, 0: unknown
  float fmax, from;
  unsigned kmin, kmax, list_n, cut_n;
  int bin_lo, bin_hi;                 // the bracket, its tokens and those above it: the same in every block
  unsigned above, upto;
  float border;                       // written by the first block, read by all
  int border_col;
  float best;                         // this block's draw
  int best_col;
  float best_z;
  float bests[8], best_zs[8];          // the first block: all blocks' draws
  int best_cols[8];
};
// the tables are read four bins at a time
static_assert(offsetof(SfShared, hist) % 16 == 0 && offsetof(SfShared, where) % 16 == 0, "bins on 16 bytes");

// A block's columns of a row.
template <typename T>
struct SfRow {
  const T* x;
  int v0, v1;
  bool vec;
  float cap;  // the quotients of larger logits are not finite
  float t;    // what logits are divided by: the temperature, or 1 where they stay as they are
  float top;  // and what none is above then
  __device__ __forceinline__ float clean(float y) const { return sf_clean1(t == 1.f ? y : __fdiv_rn(y, t), top); }
  // f(logit over t, column) over the block's columns, until stop() says so; RAW: logits as they are
  template <bool RAW = false, typename F, typename G>
  __device__ __forceinline__ void each(F f, G stop) const {
    constexpr int N = 16 / sizeof(T);
    int i = v0 + threadIdx.x;
    if (vec) {
      constexpr int U = SF_BATCH / N;
      const int n1 = v1 / N;  // v0 is a multiple of N
#pragma unroll 1
      for (int at = v0 / N + threadIdx.x; at < n1; at += U * SF_THREADS) {
        if (stop()) return;
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (at + j * SF_THREADS < n1) u[j] = reinterpret_cast<const uint4*>(x)[at + j * SF_THREADS];
#pragma unroll
        for (int j = 0; j < U; ++j) {
          if (at + j * SF_THREADS >= n1) break;
          float y[N];
          sf_unpack<T>(u[j], y);
          if (!RAW) {
#pragma unroll
            for (int k = 0; k < N; k += 4) {
              if (t == 1.f) {
#pragma unroll
                for (int e = k; e < k + 4; ++e) y[e] = sf_clean1(y[e], top);
              } else {
                const float4 z = sf_over(make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]), t);
                y[k] = z.x;
                y[k + 1] = z.y;
                y[k + 2] = z.z;
                y[k + 3] = z.w;
              }
            }
          }
#pragma unroll
          for (int k = 0; k < N; ++k) f(y[k], (at + j * SF_THREADS) * N + k);
        }
      }
      i = n1 * N + threadIdx.x;
    }
#pragma unroll 1
    for (; i < v1; i += SF_THREADS) {
      if (stop()) return;
      f(RAW ? sf_load(x, i) : clean(sf_load(x, i)), i);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each(f, [] { return false; });
  }
  // f(logits, first column) over the block's vectors of N logits (or 1), as they are
  template <typename F>
  __device__ __forceinline__ void each_vector(F f) const {
    constexpr int N = 16 / sizeof(T);
    int i = v0 + threadIdx.x;
    if (vec) {
      constexpr int U = SF_BATCH / N;
      const int n1 = v1 / N;
#pragma unroll 1
      for (int at = v0 / N + threadIdx.x; at < n1; at += U * SF_THREADS) {
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (at + j * SF_THREADS < n1) u[j] = reinterpret_cast<const uint4*>(x)[at + j * SF_THREADS];
#pragma unroll
        for (int j = 0; j < U; ++j) {
          if (at + j * SF_THREADS >= n1) break;
          float y[N];
          sf_unpack<T>(u[j], y);
          f(y, (at + j * SF_THREADS) * N);
        }
      }
      i = n1 * N + threadIdx.x;
    }
#pragma unroll 1
    for (; i < v1; i += SF_THREADS) {
      float y[1] = {sf_load(x, i)};
      f(y, i);
    }
  }
  // The same, small instead of fast: for what rows hardly ever need.
  template <typename F>
  __device__ __forceinline__ void each_slowly(F f) const {
#pragma unroll 1
    for (int i = v0 + threadIdx.x; i < v1; i += SF_THREADS) f(clean(sf_load(x, i)), i);
  }
};

__device__ __forceinline__ double sf_block_sum(double v, SfShared& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.red[0][threadIdx.x >> 5] = v;
  __syncthreads();
  double all = s.red[0][threadIdx.x & (SF_WARPS - 1)];  // one order in every warp
#pragma unroll
  for (int o = SF_WARPS / 2; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  return all;
}
__device__ __forceinline__ unsigned long long sf_block_count(unsigned long long v, SfShared& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.sum[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long all = s.sum[threadIdx.x & (SF_WARPS - 1)];
#pragma unroll
  for (int o = SF_WARPS / 2; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  return all;
}
// Inclusive prefixes over the threads of a block.
template <int N>
__device__ __forceinline__ void sf_block_prefix(double (&v)[N], SfShared& s) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, v[n], o);
      if (lane >= o) v[n] += x;
    }
  __syncthreads();
  if (lane == 31)
#pragma unroll
    for (int n = 0; n < N; ++n) s.red[n][wid] = v[n];
  __syncthreads();
  for (int w = 0; w < wid; ++w)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += s.red[n][w];
}

// One step of a bitonic sort between the lanes of a warp: `up` says whether the run that the lane is in ascends.
template <int J>
__device__ __forceinline__ void sf_sort_step(unsigned long long& x, bool up) {
  const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, J);
  if ((x > y) == (((threadIdx.x & J) == 0) == up)) x = y;
}
// Sorts n <= SF_THREADS entries ascending, one in a register of each thread of as many warps as it takes; `at` has room for the
// next power of two.
__device__ __noinline__ void sf_sort_few(unsigned long long* at, int n) {
  int size = 32;
  while (size < n) size <<= 1;
  const int i = threadIdx.x;
  __syncthreads();
  if (i < size) {
    unsigned long long x = i < n ? at[i] : ~0ull;
    sf_sort_step<1>(x, (i & 2) == 0);
    sf_sort_step<2>(x, (i & 4) == 0);
    sf_sort_step<1>(x, (i & 4) == 0);
    sf_sort_step<4>(x, (i & 8) == 0);
    sf_sort_step<2>(x, (i & 8) == 0);
    sf_sort_step<1>(x, (i & 8) == 0);
    sf_sort_step<8>(x, (i & 16) == 0);
    sf_sort_step<4>(x, (i & 16) == 0);
    sf_sort_step<2>(x, (i & 16) == 0);
    sf_sort_step<1>(x, (i & 16) == 0);
#pragma unroll 1
    for (int k = 32; k <= size; k <<= 1) {
      const bool up = (i & k) == 0;
#pragma unroll 1
      for (int j = k >> 1; j >= 32; j >>= 1) {
        at[i] = x;
        asm volatile("bar.sync 1, %0;" ::"r"(size) : "memory");
        const unsigned long long y = at[i ^ j];
        if ((x > y) == (((i & j) == 0) == up)) x = y;
        asm volatile("bar.sync 1, %0;" ::"r"(size) : "memory");
      }
      sf_sort_step<16>(x, up);
      sf_sort_step<8>(x, up);
      sf_sort_step<4>(x, up);
      sf_sort_step<2>(x, up);
      sf_sort_step<1>(x, up);
    }
    at[i] = x;
  }
  __syncthreads();
}
// Sorts n entries ascending; `at` has room for the next power of two.  As many warps as it takes pairs for work on it: the
// others wait once, at the end.
__device__ __noinline__ void sf_sort(unsigned long long* at, int n) {
  int size = 2;
  while (size < n) size <<= 1;
  const int workers = min(SF_THREADS, max(32, size / 2));
  __syncthreads();
  if (threadIdx.x < workers) {
    auto meet = [&] {
      if (workers == 32) __syncwarp();
      else asm volatile("bar.sync 1, %0;" ::"r"(workers) : "memory");
    };
    for (int i = n + threadIdx.x; i < size; i += workers) at[i] = ~0ull;
    meet();
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        for (int i = threadIdx.x; i < size / 2; i += workers) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const unsigned long long x = at[a], y = at[b];
          if ((x > y) == ((a & k) == 0)) { at[a] = y; at[b] = x; }
        }
        meet();
      }
  }
  __syncthreads();
}
__device__ __forceinline__ float sf_entry_x(unsigned long long e) { return sf_unkey(~(unsigned)(e >> 32)); }

// The better of two draws: the larger key, then the lower column; col < 0: none.
__device__ __forceinline__ void sf_better(float& best, int& col, float& z, float ob, int oc, float oz) {
  if (oc >= 0 && (col < 0 || ob > best || (ob == best && oc < col))) { best = ob; col = oc; z = oz; }
}
__device__ __forceinline__ void sf_block_best(float& best, int& col, float& z, SfShared& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ob = __shfl_xor_sync(0xffffffffu, best, o), oz = __shfl_xor_sync(0xffffffffu, z, o);
    const int oc = __shfl_xor_sync(0xffffffffu, col, o);
    sf_better(best, col, z, ob, oc, oz);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    s.warp_best[threadIdx.x >> 5] = best;
    s.warp_col[threadIdx.x >> 5] = col;
    s.warp_z[threadIdx.x >> 5] = z;
  }
  __syncthreads();
  best = s.warp_best[threadIdx.x & (SF_WARPS - 1)];
  col = s.warp_col[threadIdx.x & (SF_WARPS - 1)];
  z = s.warp_z[threadIdx.x & (SF_WARPS - 1)];
#pragma unroll
  for (int o = SF_WARPS / 2; o > 0; o >>= 1) {
    const float ob = __shfl_xor_sync(0xffffffffu, best, o), oz = __shfl_xor_sync(0xffffffffu, z, o);
    const int oc = __shfl_xor_sync(0xffffffffu, col, o);
    sf_better(best, col, z, ob, oc, oz);
  }
}

template <typename T>
struct SfSampler {
  SfShared& s;
  cg::cluster_group cluster;
  const SampleArgs& a;
  SfRow<T> r;
  int C, rank, row, tid;
  // The temperature of what is compared (logits, or with `divided` z, in lists and in run()): 1 once that is z.
  // c: of a distance to the maximum, the exponent of 2.
  float temperature, c;
  float xmax, zmax;
  float step;             // bins of the linear histogram per unit of the logits
  uint32_t word;
  bool greedy, as_sampler;  // the latter: random numbers as trlb_sample makes them
  bool divided;             // the order of the logits is not that of z
  SfShared* lead;

  __device__ __forceinline__ SfShared* of(int c) { return cluster.map_shared_rank(&s, c); }
  // What a pass needs of a row, by value: it stays in registers where the members of this object do not.
  struct Pass {
    SfRow<T> r;
    float xmax, c, step;
    // 2^y by one instruction: off by 2^-22 at most; what is below 2^-126 counts as nothing
    __device__ __forceinline__ float weight(float x) const { return fast_exp2((x - xmax) * c); }
    __device__ __forceinline__ int linear_bin(float x) const { return (int)fminf((xmax - x) * step, (float)(SF_BINS - 1)); }
  };
  __device__ __forceinline__ Pass pass() const { return {r, xmax, c, step}; }
  __device__ __forceinline__ float weight(float x) const { return exp2f((x - xmax) * c); }
  __device__ __forceinline__ float noise(uint32_t h) const { return as_sampler ? sf_gumbel_as_sampler(h) : sf_gumbel(h); }
  __device__ __forceinline__ float quotient(float x) const { return sf_quotient(x, temperature); }
  // Whether the row's logits are divided as they are read.
  __device__ __forceinline__ void read_divided(bool yes) {
    divided = yes;
    r.t = yes ? temperature : 1.f;
    r.top = yes ? SF_MAX : INFINITY;
  }
  // From here on what is compared is z.
  __device__ __forceinline__ void to_z() {
    temperature = 1.f;
    c = SF_LOG2E;
    xmax = zmax;
  }
  // The smallest logit whose quotient is at least z.
  __device__ __noinline__ float least_of(float z) const {
    if (temperature == 1.f) return z;
    if (!(z >= -SF_MAX)) return -SF_MAX;
    float x = fminf(fmaxf((float)((double)z * (double)temperature), -SF_MAX), SF_MAX);
    for (int i = 0; i < 4 && quotient(x) < z; ++i) x = nextafterf(x, INFINITY);
    for (int i = 0; i < 4 && quotient(nextafterf(x, -INFINITY)) >= z; ++i) x = nextafterf(x, -INFINITY);
    if (quotient(x) >= z && quotient(nextafterf(x, -INFINITY)) < z) return x;
    uint32_t lo = sf_key(-INFINITY), hi = sf_key(INFINITY);  // among the denormal numbers many logits have one quotient
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (quotient(sf_unkey(mid)) >= z) hi = mid;
      else lo = mid;
    }
    return sf_unkey(hi);
  }
  // x moved down, and up, to a logit at which a z begins.
  __device__ __forceinline__ float class_from(float x) const { return sizeof(T) == 2 ? x : least_of(quotient(x)); }
  __device__ __forceinline__ float class_above(float x) const {
    if (sizeof(T) == 2) return x;
    const float z = quotient(x), from = least_of(z);
    return from >= x ? from : least_of(nextafterf(z, INFINITY));
  }
  // Bins that reach down to `from`, where that is not too far.
  __device__ __forceinline__ void set_step(float from) {
    const float far = (xmax - from) / temperature;
    step = (far < 31.f ? (float)(SF_BINS - 2) / fmaxf(far, 1e-3f) : 64.f) / temperature;
  }

  // Sum and maximum over the blocks of a value that each of them left in its shared memory: a lane reads a block's, so that the
  // reads are under way together; the tree of the shuffles adds them in one order.
  template <typename F>
  __device__ __forceinline__ double sum_of(F value) {
    const int lane = tid & 31;
    double v = lane < C ? value(*of(lane)) : 0.;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0);
  }
  template <typename F>
  __device__ __forceinline__ float max_of(F value) {
    const int lane = tid & 31;
    float v = lane < C ? value(*of(lane)) : -INFINITY;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return __shfl_sync(0xffffffffu, v, 0);
  }
  // Sum of a block-wide value over the cluster, in the order of the blocks.  Ends with a barrier.
  __device__ double cluster_sum(double v) {
    v = sf_block_sum(v, s);
    if (tid == 0) s.mass = v;
    cluster.sync();
    const double all = sum_of([](const SfShared& o) { return o.mass; });
    cluster.sync();
    return all;
  }
  __device__ void clear_hist() {
    for (int i = tid; i < SF_BINS; i += SF_THREADS) s.hist[i] = 0;
    __syncthreads();
  }
  // This thread's bins of the whole row.  The table may be written again behind the next barrier.
  __device__ __noinline__ void merged_bins(unsigned (&n)[SF_EACH]) {
    cluster.sync();
    merge([](const SfShared& o) { return o.hist; }, n);
  }
  template <typename F>
  __device__ __forceinline__ void merge(F table, unsigned (&n)[SF_EACH]) {
    uint4 x[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      x[b] = make_uint4(0, 0, 0, 0);
      if (b < C) x[b] = reinterpret_cast<const uint4*>(table(*of(b)))[tid];
    }
#pragma unroll
    for (int i = 0; i < SF_EACH; ++i) n[i] = 0;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      n[0] += x[b].x;
      n[1] += x[b].y;
      n[2] += x[b].z;
      n[3] += x[b].w;
    }
  }
  // Those of this block.
  __device__ void own_bins(unsigned (&n)[SF_EACH]) {
    __syncthreads();
    const uint4 x = reinterpret_cast<const uint4*>(s.hist)[tid];
    n[0] = x.x;
    n[1] = x.y;
    n[2] = x.z;
    n[3] = x.w;
    __syncthreads();
  }
  // The bin of the k-th token of the histogram.
  __device__ __noinline__ void bracket_count(const unsigned (&n)[SF_EACH], unsigned k) {
    const unsigned own = n[0] + n[1] + n[2] + n[3];
    double v[1] = {(double)own};
    sf_block_prefix(v, s);
    unsigned below = (unsigned)v[0] - own;
#pragma unroll
    for (int i = 0; i < SF_EACH; ++i) {
      if (below < k && k <= below + n[i]) {
        s.bin_lo = s.bin_hi = SF_EACH * tid + i;
        s.above = below;
        s.upto = below + n[i];
      }
      below += n[i];
    }
    __syncthreads();
  }
  // Bins between which the mass passes `goal`: the first whose upper bound of the mass up to it does, to the first whose
  // lower bound does.  hi / lo: bounds of the mass in this thread's bins; mass: what stands above the histogram.  With `keep`
  // s.cumul has the tokens up to and with each bin.
  __device__ __noinline__ void bracket_mass(const unsigned (&n)[SF_EACH], const float (&hi)[SF_EACH], const float (&lo)[SF_EACH], double mass, double goal, bool keep) {
    if (tid == 0) {
      s.bin_lo = s.bin_hi = SF_BINS - 1;
      s.above = s.upto = 0;
    }
    // 32 bits do: the bounds are apart by more than some tens of roundings
    const int lane = tid & 31, wid = tid >> 5;
    float v[2] = {hi[0] + hi[1] + hi[2] + hi[3], lo[0] + lo[1] + lo[2] + lo[3]};
    unsigned cnt = n[0] + n[1] + n[2] + n[3];
    const float own[2] = {v[0], v[1]};
    const unsigned own_n = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float x = __shfl_up_sync(0xffffffffu, v[0], o), y = __shfl_up_sync(0xffffffffu, v[1], o);
      const unsigned z = __shfl_up_sync(0xffffffffu, cnt, o);
      if (lane >= o) { v[0] += x; v[1] += y; cnt += z; }
    }
    __syncthreads();
    if (lane == 31) { s.warp_best[wid] = v[0]; s.warp_z[wid] = v[1]; s.warp_col[wid] = (int)cnt; }
    __syncthreads();
    const float up = (float)mass + warp_sum(lane < wid ? s.warp_best[lane] : 0.f) + v[0] - own[0];  // bounds before this thread's bins
    const float low = (float)mass + warp_sum(lane < wid ? s.warp_z[lane] : 0.f) + v[1] - own[1];
    const unsigned before = __reduce_add_sync(0xffffffffu, lane < wid ? (unsigned)s.warp_col[lane] : 0u);
    cnt += before - own_n;
    const float limit = (float)goal;
    float upper = up, lower = low;
    int first_up = SF_BINS - 1, first_low = SF_BINS - 1;
#pragma unroll
    for (int i = 0; i < SF_EACH; ++i) {
      upper += hi[i];
      lower += lo[i];
      if (upper * 1.00001f > limit) first_up = min(first_up, SF_EACH * tid + i);
      if (lower * 0.99999f > limit) first_low = min(first_low, SF_EACH * tid + i);
    }
    first_up = __reduce_min_sync(0xffffffffu, first_up);
    first_low = __reduce_min_sync(0xffffffffu, first_low);
    if ((tid & 31) == 0) {
      atomicMin(&s.bin_lo, first_up);
      atomicMin(&s.bin_hi, first_low);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SF_EACH; ++i) {
      if (SF_EACH * tid + i == s.bin_lo) s.above = cnt;
      cnt += n[i];
      if (SF_EACH * tid + i == s.bin_hi) s.upto = cnt;
      if (keep) s.cumul[SF_EACH * tid + i] = cnt;
    }
    __syncthreads();
  }
  // Bounds of the mass of this thread's bins of the linear histogram, from counts alone.
  __device__ void linear_bounds(const unsigned (&n)[SF_EACH], float (&hi)[SF_EACH], float (&lo)[SF_EACH]) const {
#pragma unroll
    for (int i = 0; i < SF_EACH; ++i) {
      const int bin = SF_EACH * tid + i;
      hi[i] = (float)n[i] * exp2f(-(float)bin / step * c) * 1.00001f;
      lo[i] = bin == SF_BINS - 1 ? 0.f : (float)n[i] * exp2f(-(float)(bin + 1) / step * c) * 0.99999f;
    }
  }
  // The same with the sums of the places in the bins: a token's weight is exp(-y) of the bin's upper one, y its place times the
  // bin's width, and 1 - y <= exp(-y) <= 1 - y + y^2 / 2.
  __device__ void placed_bounds(const unsigned (&n)[SF_EACH], const unsigned (&place)[SF_EACH], float (&hi)[SF_EACH], float (&lo)[SF_EACH]) const {
    const float width = c * 0.6931471805599453f / step;
#pragma unroll
    for (int i = 0; i < SF_EACH; ++i) {
      const int bin = SF_EACH * tid + i;
      const float top = exp2f(-(float)bin / step * c), y = (float)place[i] / SF_FINE * width, slack = (float)n[i] * width / SF_FINE;
      hi[i] = fminf((float)n[i], (float)n[i] - y + slack + 0.5f * width * y) * top * 1.00001f;
      lo[i] = bin == SF_BINS - 1 ? 0.f : fmaxf((float)n[i] * (1.f - width), (float)n[i] - y - slack) * top * 0.99999f;
    }
  }
  // Bounds of the mass of this thread's bins of the histogram of keys from `top` down over `span`.
  __device__ void key_bounds(const unsigned (&n)[SF_EACH], float (&hi)[SF_EACH], float (&lo)[SF_EACH], unsigned top, unsigned span, int shift) const {
#pragma unroll
    for (int i = 0; i < SF_EACH; ++i) {
      const unsigned bin = (unsigned)(SF_EACH * tid + i);
      hi[i] = lo[i] = 0.f;
      if (bin <= span >> shift) {
        hi[i] = (float)n[i] * weight(sf_unkey(top - (bin << shift))) * 1.00001f;
        lo[i] = (float)n[i] * weight(sf_unkey(top - min((bin << shift) + ((1u << shift) - 1u), span))) * 0.99999f;
      }
    }
  }
  // Lists the row's tokens that `in` takes in the first block, in no order; returns their number, 0 where the list is too short.
  template <typename F>
  __device__ __forceinline__ int gather(F in) {
    if (tid == 0) s.list_n = 0;
    __syncthreads();
    {
      SfShared& sh = s;
      const SfRow<T> q = r;
      q.each(
          [&](float x, int col) {
            if (in(x)) {
              append(sh, x, col);
            }
          },
          [&] { return *reinterpret_cast<volatile unsigned*>(&sh.list_n) > SF_LIST; });
    }
    return collect();
  }
  // The blocks' lists in the first one.
  __device__ __noinline__ int collect() {
    cluster.sync();
    const int lane = tid & 31, mine = lane < C ? (int)of(lane)->list_n : 0;
    int upto = mine;  // entries of the blocks up to this lane's
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const int n = __shfl_sync(0xffffffffu, upto, 7);
    if (n > SF_LIST) return 0;
    if (rank == 0) {
      // each warp copies part of one other block's list
      constexpr int W = SF_WARPS / 8;
      const int b = (tid >> 5) / W, part = (tid >> 5) % W;
      const int m = __shfl_sync(0xffffffffu, mine, b), at = __shfl_sync(0xffffffffu, upto, b) - m;
      if (b > 0 && b < C) {
        const unsigned long long* from = of(b)->list;
        for (int i = part * 32 + lane; i < m; i += W * 32) s.list[at + i] = from[i];
      }
      __syncthreads();
    }
    return n;
  }

  // ---- the first block alone: borders in its list of n tokens -----------------------------------------------------------
  __device__ __forceinline__ unsigned long long whole(double w) const { return (unsigned long long)(w * SF_UNIT + 0.5); }
  // Where one of n <= SF_THREADS entries stands among them: entries before it and their mass; is_k: its logit is at least that of
  // the k-th.  Up to SF_FEW each is compared with all others, by as many threads as there are for it, more are sorted: of 44 that takes 4.9 us
  // instead of 5.8, of 59 6.9 instead of 8.4, of 117 as long as sorting.
  struct Place {
    unsigned long long entry, own, before;
    unsigned rank;
    bool valid, is_k;  // valid: this thread answers for the entry
  };
  __device__ __forceinline__ unsigned long long mass_of(unsigned long long e) const { return whole((double)expf(quotient(sf_entry_x(e)) - zmax)); }
  __device__ __noinline__ Place place_of(unsigned long long* at, int n, int k) {
    Place p;
    if (n <= SF_FEW) {
      int each = SF_THREADS / SF_FEW;
      while (each < 32 && 2 * each * n <= SF_THREADS) each *= 2;
      ulonglong2* pairs = reinterpret_cast<ulonglong2*>(s.hist);
      __syncthreads();
      if (tid < n) pairs[tid] = make_ulonglong2(at[tid], mass_of(at[tid]));
      __syncthreads();
      const ulonglong2 mine = pairs[min(tid / each, n - 1)];
      p.entry = mine.x;
      p.own = mine.y;
      p.before = 0;
      p.rank = 0;
      unsigned larger = 0;
      for (int j = tid & (each - 1); j < n; j += each) {
        const ulonglong2 o = pairs[j];
        if (o.x < mine.x) {
          p.before += o.y;
          ++p.rank;
        }
        larger += (unsigned)(o.x >> 32) < (unsigned)(mine.x >> 32);
      }
      for (int o = each / 2; o > 0; o >>= 1) {
        p.before += __shfl_xor_sync(0xffffffffu, p.before, o);
        p.rank += __shfl_xor_sync(0xffffffffu, p.rank, o);
        larger += __shfl_xor_sync(0xffffffffu, larger, o);
      }
      p.valid = tid < n * each && (tid & (each - 1)) == 0;
      p.is_k = (int)larger < k;
      return p;
    }
    sf_sort_few(at, n);
    const int lane = tid & 31, wid = tid >> 5;
    p.valid = tid < n;
    p.entry = at[min(tid, n - 1)];
    p.own = p.valid ? mass_of(p.entry) : 0;
    p.rank = (unsigned)tid;
    p.is_k = k > 0 && (unsigned)(p.entry >> 32) <= (unsigned)(at[min(k, n) - 1] >> 32);
    unsigned long long upto = p.own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s.sum[wid] = upto;
    __syncthreads();
    unsigned long long others = lane < wid ? s.sum[lane & (SF_WARPS - 1)] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) others += __shfl_xor_sync(0xffffffffu, others, o);
    p.before = upto - p.own + others;
    return p;
  }
  // The border among n <= SF_THREADS entries; `above` tokens and `mass` above them.
  __device__ __noinline__ void few_border(unsigned long long* at, int n, bool by_mass, double goal, unsigned above, double mass) {
    const Place p = place_of(at, n, 0);
    bool border = p.valid;
    double kept = 0.;
    if (by_mass) {
      // the last entry before which at most `goal` stands: its successor is behind more
      kept = mass + (double)(p.before + p.own) / SF_UNIT;
      border = border && (p.rank == 0 || mass + (double)p.before / SF_UNIT <= goal) && (p.rank == n - 1 || kept > goal);
    } else {
      border = border && above + p.rank + 1 == (unsigned)goal;
    }
    if (border) {
      s.border = sf_entry_x(p.entry);
      s.border_col = by_mass ? (int)(unsigned)p.entry : 0x7fffffff;
      s.kept = kept;
    }
    __syncthreads();
  }
  // The border among n entries that are sorted.
  __device__ __noinline__ void sorted_border(const unsigned long long* at, int n, bool by_mass, double goal, unsigned above, double mass) {
    if (!by_mass) {
      if (tid == 0) {
        s.border = sf_entry_x(at[(unsigned)goal - above - 1]);
        s.border_col = 0x7fffffff;
        s.kept = 0.;
      }
      __syncthreads();
      return;
    }
    constexpr int E = SF_LIST / SF_THREADS;
    double v[1] = {0.};
    for (int e = 0; e < E; ++e) v[0] += tid * E + e < n ? (double)weight(sf_entry_x(at[tid * E + e])) : 0.;
    const double own = v[0];
    sf_block_prefix(v, s);
    if (tid == 0) s.bin_lo = 0;
    __syncthreads();
    double before = mass + (v[0] - own);
    for (int e = 0; e < E && tid * E + e < n; ++e) {
      if (before <= goal) atomicMax(&s.bin_lo, tid * E + e);
      before += (double)weight(sf_entry_x(at[tid * E + e]));
    }
    __syncthreads();
    const int last = s.bin_lo;
    before = mass + (v[0] - own);
    for (int e = 0; e < E && tid * E + e < n; ++e) {
      before += (double)weight(sf_entry_x(at[tid * E + e]));
      if (tid * E + e == last) {
        s.kept = before;
        s.border = sf_entry_x(at[last]);
        s.border_col = (int)(unsigned)at[last];
      }
    }
    __syncthreads();
  }
  // The border in the list of n tokens, `above` of them and `mass` above it: the last token before which at most `goal` of mass
  // stands (by_mass), or the goal-th token and its equals.  Leaves s.border, s.border_col and s.kept (0: unknown).
  __device__ __noinline__ void list_border(int n, bool by_mass, double goal, unsigned above, double mass) {
    if (n <= SF_THREADS) {
      few_border(s.list, n, by_mass, goal, above, mass);
      return;
    }
    unsigned lo = 0xffffffffu, hi = 0u;
    for (int i = tid; i < n; i += SF_THREADS) {
      const unsigned k = ~(unsigned)(s.list[i] >> 32);
      lo = min(lo, k);
      hi = max(hi, k);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (tid == 0) { s.kmin = 0xffffffffu; s.kmax = 0u; s.cut_n = 0; }
    clear_hist();
    if ((tid & 31) == 0) { atomicMin(&s.kmin, lo); atomicMax(&s.kmax, hi); }
    __syncthreads();
    lo = s.kmin;
    hi = s.kmax;
    int shift = 0;
    while (((hi - lo) >> shift) >= SF_BINS) ++shift;
    for (int i = tid; i < n; i += SF_THREADS) atomicAdd(&s.hist[(hi - ~(unsigned)(s.list[i] >> 32)) >> shift], 1u);
    unsigned cnt[SF_EACH];
    own_bins(cnt);
    if (by_mass) {
      float wh[SF_EACH], wl[SF_EACH];
      key_bounds(cnt, wh, wl, hi, hi - lo, shift);
      bracket_mass(cnt, wh, wl, mass, goal, false);
    } else {
      bracket_count(cnt, (unsigned)goal - above);
    }
    const unsigned b0 = (unsigned)s.bin_lo, b1 = (unsigned)s.bin_hi, a0 = s.above, around = s.upto - s.above;
    __syncthreads();
    if (around > SF_CUT) {  // (nearly) equals: in place
      sf_sort(s.list, n);
      sorted_border(s.list, n, by_mass, goal, above, mass);
      return;
    }
    unsigned long long before = 0;
    for (int i = tid; i < n; i += SF_THREADS) {
      const unsigned long long e = s.list[i];
      const unsigned bin = (hi - ~(unsigned)(e >> 32)) >> shift;
      if (bin >= b0 && bin <= b1) s.cut[atomicAdd(&s.cut_n, 1u)] = e;
      else if (bin < b0 && by_mass) before += whole((double)weight(sf_entry_x(e)));
    }
    if (by_mass) mass += (double)sf_block_count(before, s) / SF_UNIT;
    __syncthreads();
    const int m = (int)s.cut_n;
    above += a0;
    if (m <= SF_THREADS) {
      few_border(s.cut, m, by_mass, goal, above, mass);
    } else {
      sf_sort(s.cut, m);
      sorted_border(s.cut, m, by_mass, goal, above, mass);
    }
  }
  static __device__ __forceinline__ bool within(float x, int col, float border, int border_col) {
    return x > border || (x == border && col <= border_col);
  }
  // Sums and draws over the list's tokens down to the border and at least `floor`.
  __device__ __noinline__ void finish_list(int n, float border, int border_col, float floor) {
    unsigned long long sum = 0;
    float best = -INFINITY, best_z = 0.f;
    int col = -1;
    for (int i = tid; i < n; i += SF_THREADS) {
      const unsigned long long e = s.list[i];
      const float x = sf_entry_x(e);
      const int at = (int)(unsigned)e;
      if (x < floor || !within(x, at, border, border_col)) continue;
      const float z = quotient(x);
      sum += whole((double)expf(z - zmax));
      sf_better(best, col, best_z, greedy ? z : z + noise(sf_bits(word, (uint32_t)at)), at, z);
    }
    sum = sf_block_count(sum, s);
    sf_block_best(best, col, best_z, s);
    write(best_z, col, (double)sum / SF_UNIT);
  }
  __device__ void write(float z, int col, double mass) {
    if (tid == 0) {
      a.tok[row] = col;
      a.logp[row] = (float)((double)z - (double)zmax - log(mass));
    }
  }

  // ---- all blocks ----------------------------------------------------------------------------------------------------
  // What the first block found, for every block.
  __device__ __noinline__ void share_border(float& border, int& border_col, double& kept) {
    cluster.sync();
    border = lead->border;
    border_col = lead->border_col;
    kept = lead->kept;
    cluster.sync();
  }
  // The border of top-k (by_mass false: goal is a number of tokens) or top-p (goal is a mass) among the tokens that are at least
  // `floor`; with floor_mass the goal is that share of their mass.  Returns the number of entries of the first block's list if
  // that holds every token down to the border's bin (and sets goal), else 0 and the border; kept: the mass down to it, if known.
  __device__ __noinline__ int search(bool by_mass, double& goal, bool floor_mass, float floor, float& border, int& border_col, double& kept) {
    kept = 0.;
    set_step(floor);
    clear_hist();
    float part = 0.f;
    const Pass q = pass();
    {
      unsigned* hist = s.hist;
      const float from = fmaxf(floor, -SF_MAX);
      q.r.each([&](float x, int) {
        if (x >= from) {
          atomicAdd(&hist[q.linear_bin(x)], 1u);
          if (floor_mass) part += q.weight(x);
        }
      });
    }
    if (floor_mass) goal *= cluster_sum((double)part);
    unsigned n[SF_EACH];
    merged_bins(n);
    cluster.sync();
    const double limit = goal;
    if (by_mass) {
      float hi[SF_EACH], lo[SF_EACH];
      linear_bounds(n, hi, lo);
      bracket_mass(n, hi, lo, 0., limit, false);
    } else {
      double all[1] = {(double)n[0] + n[1] + n[2] + n[3]};
      sf_block_prefix(all, s);
      if (tid == SF_THREADS - 1) s.upto = (unsigned)all[0];
      __syncthreads();
      const unsigned finite = s.upto;
      __syncthreads();
      if (goal > (double)finite) {  // fewer tokens than k: all are kept
        border = -INFINITY;
        border_col = 0x7fffffff;
        return 0;
      }
      bracket_count(n, (unsigned)goal);
    }
    const int b0 = s.bin_lo, b1 = s.bin_hi;
    unsigned above = s.above, upto = s.upto;
    __syncthreads();
    const float from = fmaxf(floor, -SF_MAX);
    if (upto <= SF_LIST) return gather([&](float x) { return x >= from && q.linear_bin(x) <= b1; });
    auto member = [&](float x) {
      const int b = q.linear_bin(x);
      return x >= from && b >= b0 && b <= b1;
    };
    auto over = [&](float x) { return x >= -SF_MAX && q.linear_bin(x) < b0; };
    double mass = 0.;
    part = 0.f;
    if (upto - above <= SF_LIST) {
      const int m = gather([&](float x) {
        const int b = q.linear_bin(x);
        if (by_mass && b < b0) part += q.weight(x);
        return x >= from && b >= b0 && b <= b1;
      });
      if (by_mass) mass = cluster_sum((double)part);
      if (rank == 0) {
        list_border(m, by_mass, limit, above, mass);
      }
      share_border(border, border_col, kept);
      return 0;
    }
    // keys of the bracket, and the mass above it
    unsigned kmin = 0xffffffffu, kmax = 0u;
    r.each_slowly([&](float x, int) {
      if (member(x)) {
        kmin = min(kmin, sf_key(x));
        kmax = max(kmax, sf_key(x));
      } else if (over(x)) {
        part += weight(x);
      }
    });
    kmin = __reduce_min_sync(0xffffffffu, kmin);
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (tid == 0) { s.kmin = 0xffffffffu; s.kmax = 0u; }
    __syncthreads();
    if ((tid & 31) == 0) { atomicMin(&s.kmin, kmin); atomicMax(&s.kmax, kmax); }
    mass = cluster_sum((double)part);  // its barriers show kmin and kmax, too
    for (int b = 0; b < C; ++b) {
      kmin = min(kmin, of(b)->kmin);
      kmax = max(kmax, of(b)->kmax);
    }
    cluster.sync();
    // All tokens with keys in [kmin, kmax] are the bracket's: the bins are intervals of the logits.  Each turn leaves an
    // interval of one bin's width, so there are three at most.
    while (upto - above > SF_LIST && kmin < kmax) {
      int shift = 0;
      while (((kmax - kmin) >> shift) >= SF_BINS) ++shift;
      const unsigned top = kmax, span = kmax - kmin;
      clear_hist();
      r.each_slowly([&](float x, int) {
        const unsigned k = sf_key(x);
        if (k >= kmin && k <= top) atomicAdd(&s.hist[(top - k) >> shift], 1u);
      });
      merged_bins(n);
      cluster.sync();
      unsigned c0, c1, a0, a1;  // the bracket's bins; tokens of the interval above it, and up to its end
      if (by_mass) {
        float hi[SF_EACH], lo[SF_EACH];
        key_bounds(n, hi, lo, top, span, shift);
        bracket_mass(n, hi, lo, mass, limit, true);
        c0 = (unsigned)s.bin_lo, c1 = (unsigned)s.bin_hi, a0 = s.above, a1 = s.upto;
        __syncthreads();
        auto between = [&](unsigned from, unsigned to) {  // exact mass of a run of bins
          float sum = 0.f;
          r.each_slowly([&](float x, int) {
            const unsigned k = sf_key(x);
            if (k >= kmin && k <= top && (top - k) >> shift >= from && (top - k) >> shift <= to) sum += weight(x);
          });
          return cluster_sum((double)sum);
        };
        if (c0 > 0) mass += between(0, c0 - 1);
        // the bounds leave several bins only where the goal is within their margin of a bin's end
        while (c0 < c1 && a1 - a0 > SF_LIST) {
          const unsigned mid = (c0 + c1) / 2, am = s.cumul[mid];
          const double here = between(c0, mid);
          if (mass + here <= limit && am < a1) {
            mass += here;
            a0 = am;
            c0 = mid + 1;
          } else {
            c1 = mid;
            a1 = am;
          }
        }
      } else {
        bracket_count(n, (unsigned)goal - above);
        c0 = c1 = (unsigned)s.bin_lo, a0 = s.above, a1 = s.upto;
        __syncthreads();
      }
      kmax = top - min(c0 << shift, span);
      kmin = top - min((c1 << shift) + ((1u << shift) - 1u), span);
      upto = above + a1;
      above += a0;
    }
    if (upto - above <= SF_LIST) {
      const int m = gather([&](float x) { const unsigned k = sf_key(x); return k >= kmin && k <= kmax; });
      if (rank == 0) {
        list_border(m, by_mass, limit, above, mass);
      }
      share_border(border, border_col, kept);
      return 0;
    }
    // more equals than the list holds
    border = sf_unkey(kmax);
    border_col = 0x7fffffff;
    if (by_mass) {
      const double w = (double)weight(border), equals = (double)(upto - above);
      const double fit = w > 0. ? ::floor((limit - mass) / w) + 1. : equals;  // how many of them are kept
      if (fit < equals) border_col = column_of(kmax, (unsigned)fmax(1., fit));
    }
    return 0;
  }
  // The column of the n-th token (in the order of the columns, from 1) whose key is `key`.
  __device__ __noinline__ int column_of(unsigned key, unsigned n) {
    int width = (a.V + SF_BINS - 1) / SF_BINS;
    clear_hist();
    r.each_slowly([&](float x, int col) { if (sf_key(x) == key) atomicAdd(&s.hist[col / width], 1u); });
    unsigned m[SF_EACH];
    merged_bins(m);
    cluster.sync();
    bracket_count(m, n);
    const int bin = s.bin_lo;
    const unsigned before = s.above;
    __syncthreads();
    if (rank == 0 && tid == 0) {  // some hundred columns: one thread counts its way through them
      const int lo = bin * width, hi = min(a.V, lo + width);
      unsigned count = before;
      int found = hi - 1;
      for (int i = lo; i < hi; ++i)
        if (sf_key(r.clean(sf_load(r.x, i))) == key && ++count == n) { found = i; break; }
      s.border_col = found;
    }
    cluster.sync();
    const int col = lead->border_col;
    cluster.sync();
    return col;
  }

  // The draw among the list's tokens down to the border and what the blocks drew above the list; `mass` of all of it.
  __device__ __noinline__ void finish_blocks(int n, float border, int border_col, double mass) {
    float best = -INFINITY, best_z = 0.f;
    int col = -1;
    for (int i = tid; i < n; i += SF_THREADS) {
      const unsigned long long e = s.list[i];
      const float x = sf_entry_x(e);
      const int at = (int)(unsigned)e;
      if (!within(x, at, border, border_col)) continue;
      const float z = quotient(x);
      sf_better(best, col, best_z, z + noise(sf_bits(word, (uint32_t)at)), at, z);
    }
    if (tid < C) sf_better(best, col, best_z, s.bests[tid], s.best_cols[tid], s.best_zs[tid]);
    sf_block_best(best, col, best_z, s);
    if ((double)best < (double)zmax + (double)logf((float)mass) - 2.999) {  // once in 10^8 rows: without the shortcut of the draws
      SfRow<T> q = r;
      q.v0 = 0;
      q.v1 = a.V;
      best = -INFINITY;
      col = -1;
      q.each_slowly([&](float x, int at) {
        if (x >= -SF_MAX && within(x, at, border, border_col)) {
          const float z = quotient(x);
          sf_better(best, col, best_z, z + noise(sf_bits(word, (uint32_t)at)), at, z);
        }
      });
      sf_block_best(best, col, best_z, s);
    }
    write(best_z, col, mass);
  }

  // The first block has what it needs of the others, which leave: their places are free for the next row.
  __device__ __forceinline__ void release(bool draws) {
    if (draws && rank == 0 && tid < C) {
      s.bests[tid] = of(tid)->best;
      s.best_cols[tid] = of(tid)->best_col;
      s.best_zs[tid] = of(tid)->best_z;
    }
    cluster.sync();
  }

  // The block's columns, HELD: in shared memory, `vecs` vectors, of which a thread reads what it has written; else read again for
  // each pass.  False where the row needs run().
  template <bool HELD>
  __device__ __forceinline__ bool fast(uint4* data, int vecs) {
    constexpr int N = 16 / sizeof(T);
    const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;
    const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
    const bool by_k = top_k > 0 && top_k < a.V, by_p = top_p < 1.f;
    if (!(temperature <= SF_HIGH)) return false;
    // Sums over many tokens are of the weights of undivided logits.  At low temperatures only those of the tokens that have any.
    const bool low = temperature < SF_LOW;
    if (by_k && !low && top_k > min(SF_LIST / 4, C * SF_THREADS / 2)) return false;  // too many for the lists
    const int first = r.v0;
    // A thread's maximum and, where it counts, the mass relative to it.
    float mine = -INFINITY, part = 0.f;
    const float per_unit = c;
    auto take = [&](auto& y) {
      constexpr int M = sizeof(y) / sizeof(float);
      float top = y[0];
#pragma unroll
      for (int k = 1; k < M; ++k) top = fmaxf(top, y[k]);
      if (by_k || low) {
        mine = fmaxf(mine, top);
        return;
      }
      if (top > mine) {  // rare after the first few
        part *= fast_exp2((mine - top) * per_unit);
        mine = top;
      }
      if (mine > -INFINITY)
#pragma unroll
        for (int k = 0; k < M; ++k) part += fast_exp2((y[k] - mine) * per_unit);
    };
    if constexpr (!HELD) {
      // what is NaN or has no finite quotient spoils the maximum, and the row: run() cleans each logit
      const SfRow<T> q = r;
      bool fine = true;
      q.each_vector([&](auto& y, int) {
#pragma unroll
        for (int k = 0; k < (int)(sizeof(y) / sizeof(float)); ++k) fine = fine && y[k] <= q.cap;
        take(y);
      });
      if (!fine) mine = INFINITY;
    } else {
      const SfRow<T> q = r;
#pragma unroll 4
      for (int v = tid; v < vecs; v += SF_THREADS) {
        const int at = first + v * N;
        uint4 u;
        if (q.vec && at + N <= q.v1) {
          u = *reinterpret_cast<const uint4*>(q.x + at);
        } else {
          uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const T y = at + k < q.v1 ? q.x[at + k] : sf_lowest<T>();
            if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(y);
            else w[k / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(&y) << (16 * (k & 1));
          }
          u = make_uint4(w[0], w[1], w[2], w[3]);
        }
        sf_clean<T>(u);
        float y[N];
        sf_unpack<T>(u, y);
        take(y);
        data[v] = u;
      }
      // what has no finite quotient (of a narrow type: infinities, beside its largest numbers) spoils the row here, too
      if (mine > q.cap) mine = INFINITY;
    }
    auto each_until = [&](auto f, auto stop) {
      if constexpr (HELD) {
#pragma unroll 1
        for (int v = tid; v < vecs; v += SF_THREADS) {
          if (stop()) return;
          float y[N];
          sf_unpack<T>(data[v], y);
#pragma unroll
          for (int k = 0; k < N; ++k) f(y[k], first + v * N + k);
        }
      } else {
        const SfRow<T> q = r;
        q.template each<true>(f, stop);
      }
    };
    auto each = [&](auto f) { each_until(f, [] { return false; }); };
    auto each_vector = [&](auto f) {
      if constexpr (HELD) {
#pragma unroll 1
        for (int v = tid; v < vecs; v += SF_THREADS) {
          float y[N];
          sf_unpack<T>(data[v], y);
          f(y, first + v * N);
        }
      } else {
        const SfRow<T> q = r;
        q.each_vector(f);
      }
    };
    SfShared& sh = s;
    // ---- the maximum of the block, the smallest of its threads' ----
    const int lane = tid & 31, wid = tid >> 5;
    const float wmax = warp_max(mine), wmin = -warp_max(mine == -INFINITY ? -INFINITY : -mine);
    if (lane == 0) { sh.red[0][wid] = wmax; sh.red[1][wid] = wmin; }
    if (tid == 0) { sh.list_n = 0; sh.bin_lo = SF_BINS; }
    for (int i = tid; i < SF_BINS; i += SF_THREADS) sh.hist[i] = sh.where[i] = 0;
    __syncthreads();
    float bmax = lane < SF_WARPS ? (float)sh.red[0][lane] : -INFINITY, bmin = lane < SF_WARPS ? (float)sh.red[1][lane] : INFINITY;
    bmax = warp_max(bmax);
    bmin = -warp_max(-bmin);
    if (by_k || low) {
      // A k-th part of the blocks' number: as many threads of each block have a maximum of at least `from`, so that k logits of
      // the row are at least the smallest of the blocks' numbers.
      const unsigned share = (unsigned)((top_k + C - 1) / C);
      float from = -SF_MAX;  // all, where fewer threads have any
      const float scale = (float)(SF_BINS - 2) / (bmax - bmin);
      if (scale < 1e30f && !low) {  // false also where the block has none or all maxima are equal
        if (mine > -INFINITY) atomicAdd(&sh.hist[(int)fminf((bmax - mine) * scale, (float)(SF_BINS - 1))], 1u);
        unsigned h[SF_EACH];
        own_bins(h);
        bracket_count(h, share);
        if (sh.bin_lo < SF_BINS - 1) from = fmaxf(from, bmax - (float)(sh.bin_lo + 1) / scale * 1.000001f);  // a little below the bin's end
      }
      if (tid == 0) { sh.fmax = bmax; sh.from = from; }
      cluster.sync();
      xmax = max_of([](const SfShared& o) { return o.fmax; });
      zmax = quotient(xmax);
      if (xmax == INFINITY || zmax == -INFINITY) return false;
      from = -max_of([](const SfShared& o) { return -o.from; });
      // 104 below the largest z a weight is below 2^-149, and no noise (of -3.2 to 23) makes up for that
      if (low) from = fmaxf(-SF_MAX, xmax - 105.f * temperature);
      from = class_from(from);
      each([&](float x, int col) {
        if (x >= from) append(sh, x, col);
      });
      const int n = collect();
      if (n == 0) return false;  // none at all, or too many
      if (n < top_k && !low) return false;
      release(false);
      if (rank == 0) {
        if (sizeof(T) == 4 || low) divide_list(n);
        top_k_of_list(n, by_k ? min(top_k, n) : n, by_p, top_p, min_p > 0.f ? least_of(least_kept(min_p)) : -INFINITY);
      }
      return true;
    }
    // ---- the mass relative to the block's maximum, then that of the row ----
    double total;
    {
      const double sum = sf_block_sum(mine > -INFINITY ? (double)(part * fast_exp2((mine - bmax) * per_unit)) : 0., sh);
      if (tid == 0) { sh.fmax = bmax; sh.sums[0] = sum; }
      cluster.sync();
      xmax = max_of([](const SfShared& o) { return o.fmax; });
      if (xmax == -INFINITY || xmax == INFINITY) return false;
      zmax = quotient(xmax);
      if (zmax == -INFINITY) return false;
      total = sum_of([&](const SfShared& o) { return o.fmax > -INFINITY ? o.sums[0] * (double)exp2f((o.fmax - xmax) * c) : 0.; });
    }
    const Pass q = pass();
    const float floor_z = min_p > 0.f ? least_kept(min_p) : -INFINITY, floor = min_p > 0.f ? least_of(floor_z) : -INFINITY;
    const float list_floor = sizeof(T) == 4 ? floor_z : floor;
    const double goal = by_p ? fmax(0., (double)top_p * total) : 0.;
    float from = -SF_MAX;
    // ---- top-p ----
    if (by_p) {
      // lighter tokens than this together have less than what top-p leaves out; a little is added for the sums' rounding
      const double least = (1. - (double)top_p - 2e-5) * total / a.V;
      if (!(least > 0.)) return false;
      from = class_from(fmaxf(-SF_MAX, xmax + (logf((float)least) - 1e-3f) * temperature));
    }
    if (by_p && goal < SF_LIST / 16) {
      // twice a block's part of the list says that there are too many, without a look at the rest
      const unsigned most = (unsigned)min(SF_LIST, 2 * SF_LIST / C);
      each_until(
          [&](float x, int col) {
            if (x >= from) append(sh, listed(x), col);
          },
          [&] { return *reinterpret_cast<volatile unsigned*>(&sh.list_n) > most; });
      __syncthreads();
      if (tid == 0 && sh.list_n > most) sh.list_n = SF_LIST + 1;
      const int n = collect();
      if (n > 0) {
        release(false);
        if (rank == 0) {
          if (sizeof(T) == 4) to_z();
          const int m = n > SF_FEW ? thin_out(n, goal, total) : n;
          if (m <= SF_THREADS) {
            finish_few(m, 0, 0., goal, list_floor);
          } else {
            list_border(m, true, goal, 0, 0.);
            finish_list(m, sh.border, sh.border_col, list_floor);
          }
        }
        return true;
      }
      cluster.sync();  // the numbers of the lists have been read
      if (tid == 0) sh.list_n = 0;
    }
    // ---- min-p: either all that it keeps is within top-p, or top-p keeps less and min-p changes nothing ----
    bool all = !by_p;
    double floor_mass = total;
    if (floor > -INFINITY) {
      float part = 0.f;
      each([&](float x, int) { part += x >= floor ? q.weight(x) : 0.f; });
      const double sum = sf_block_sum((double)part, sh);
      if (tid == 0) sh.sums[1] = sum;
      cluster.sync();
      floor_mass = sum_of([](const SfShared& o) { return o.sums[1]; });
      all = all || floor_mass <= goal;
    }
    if (all) {
      draw(each_vector, q, floor_mass, floor);
      cluster.sync();
      release(true);
      if (rank == 0) {
        if (sizeof(T) == 4) to_z();
        finish_blocks(0, fmaxf(list_floor, -SF_MAX), 0x7fffffff, floor_mass);
      }
      return true;
    }
    set_step(from);
    const Pass h = pass();
    each([&](float x, int) {
      if (x >= from) {
        // bin and place in it: the whole number and the fraction of linear_bin's quotient; the last bin has all that is further
        const unsigned y = (unsigned)fminf((h.xmax - x) * h.step * SF_FINE, SF_BINS * SF_FINE - 1.f);
        atomicAdd(&sh.hist[y / (unsigned)SF_FINE], 1u);
        atomicAdd(&sh.where[y / (unsigned)SF_FINE], y % (unsigned)SF_FINE);
      }
    });
    cluster.sync();
    if (rank == 0) {  // one block's reads of all tables are faster than those of eight
      unsigned n[SF_EACH], place[SF_EACH];
      merge([](const SfShared& o) { return o.hist; }, n);
      merge([](const SfShared& o) { return o.where; }, place);
      float hi[SF_EACH], lo[SF_EACH];
      placed_bounds(n, place, hi, lo);
      bracket_mass(n, hi, lo, 0., goal, false);
    }
    cluster.sync();
    const int b0 = lead->bin_lo, b1 = lead->bin_hi;
    const unsigned above = lead->above;
    if (lead->upto - above > SF_LIST) return false;
    // above the bracket: the mass, and the draw (at least `goal` is kept); the bracket: listed
    {
      Draw d = {(float)(20.0855369 * 1.001 / goal), temperature, word, as_sampler, 0.f, -INFINITY, 0.f, -1};
      // From `sure` on a logit is in a bin above the bracket, below `last` in one behind it: the bins' ends, moved by more than the
      // rounding of linear_bin() (2^-22 of the distance), then to where a z begins.  So the list holds the bracket and the few
      // logits beside it; what is kept for sure has less mass than the goal, all of it with the list's more.
      const double bin = 1. / (double)h.step;
      const float sure = b0 > 0 ? class_above(__double2float_ru((double)h.xmax - b0 * bin * (1. - 1e-6))) : INFINITY;
      const float last = b1 < SF_BINS - 1 ? fmaxf(from, class_from(__double2float_rd((double)h.xmax - (b1 + 1) * bin * (1. + 1e-6)))) : from;
      each_vector([&](auto& x, int col) {
        constexpr int M = sizeof(x) / sizeof(float);
        unsigned keep = 0, list = 0;
#pragma unroll
        for (int k = 0; k < M; ++k) {
          keep |= (x[k] >= sure ? 1u : 0u) << k;
          list |= (x[k] >= last ? 1u : 0u) << k;
        }
        list &= ~keep;
        if (list) {
#pragma unroll
          for (int k = 0; k < M; ++k)
            if (list >> k & 1) append(sh, listed(x[k]), col + k);
        }
        if (keep) consider_vector(h, d, x, col, keep);
      });
      const double sum = sf_block_sum((double)d.part, sh);
      sf_block_best(d.top, d.at, d.top_z, sh);
      if (tid == 0) {
        sh.sums[1] = sum;
        sh.best = d.top;
        sh.best_col = d.at;
        sh.best_z = d.top_z;
      }
    }
    const int n = collect();
    if (n == 0) return false;  // too many equals at the bracket's ends
    const double mass = sum_of([](const SfShared& o) { return o.sums[1]; });
    release(true);
    if (rank == 0) {
      if (sizeof(T) == 4) to_z();
      list_border(n, true, goal, above, mass);
      finish_blocks(n, sh.border, sh.border_col, sh.kept);
    }
    return true;
  }
  static __device__ __forceinline__ void append(SfShared& sh, float x, int col) {
    const unsigned i = atomicAdd(&sh.list_n, 1u);
    if (i < SF_LIST) sh.list[i] = (unsigned long long)(~sf_key(x + 0.f)) << 32 | (unsigned)col;
  }
  // One token's chance in a draw.  The largest z - log(-log u) of the kept tokens is lse + a Gumbel variate, which is below
  // lse - 3 once in 10^8 rows.  A token reaches K = lse - 3 only if -log u <= exp(z - K), and -log u >= 1 - u: most are out
  // after their random bits.
  static __device__ __forceinline__ void consider(float x, int col, float weight, float reach, float t, uint32_t word, bool most,
                                                  bool as_sampler, float& top, int& at, float& top_z) {
    float z = x, k = x;
    if (!most) {
      const uint32_t h = sf_bits(word, (uint32_t)col);
      // 1 - u in [0, 1), its bits set behind a one; the margin is for the bits cut off and, as_sampler, for what 24 bits and fast
      // logarithms may make of it
      if (__uint_as_float(0x3f800000u | ~h >> 9) > fmaf(reach, weight, as_sampler ? 1.f + 2e-6f : 1.f + 3e-7f)) return;
      z = sf_quotient(x, t);
      k = z + (as_sampler ? sf_gumbel_as_sampler(h) : sf_gumbel(h));
    }
    if (at < 0 || k > top || (k == top && col < at)) { top = k; at = col; top_z = z; }
  }
  // The same for those of a vector's logits x[] that `keep` names, from column col on, and their mass.  All their random bits are
  // made before the first branch, so that the eight chains run beside each other.
  struct Draw {
    float reach, t;
    uint32_t word;
    bool as;
    float part, top, top_z;
    int at;
  };
  template <int M>
  static __device__ __forceinline__ void consider_vector(const Pass& q, Draw& d, const float (&x)[M], int col, unsigned keep) {
    const float margin = d.as ? 1.f + 2e-6f : 1.f + 3e-7f;
    unsigned maybe = 0;
#pragma unroll
    for (int k = 0; k < M; ++k) {
      const bool in = keep >> k & 1;
      const float w = in ? q.weight(x[k]) : 0.f;
      const uint32_t h = sf_bits(d.word, (uint32_t)(col + k));
      d.part += w;
      if (in && !(__uint_as_float(0x3f800000u | ~h >> 9) > fmaf(d.reach, w, margin))) maybe |= 1u << k;
    }
    if (maybe) {
#pragma unroll
      for (int k = 0; k < M; ++k)
        if (maybe >> k & 1) consider(x[k], col + k, INFINITY, INFINITY, d.t, d.word, false, d.as, d.top, d.at, d.top_z);
    }
  }
  // This block's draw among its tokens of at least `floor`.
  template <typename E>
  __device__ __forceinline__ void draw(E each_vector, const Pass& q, double mass, float floor) {
    const float from = fmaxf(floor, -SF_MAX);
    Draw d = {(float)(20.0855369 * 1.001 / mass), temperature, word, as_sampler, 0.f, -INFINITY, 0.f, -1};
    each_vector([&](auto& x, int col) {
      constexpr int M = sizeof(x) / sizeof(float);
      unsigned keep = 0;
#pragma unroll
      for (int k = 0; k < M; ++k) keep |= (x[k] >= from ? 1u : 0u) << k;
      if (keep) consider_vector(q, d, x, col, keep);
    });
    sf_block_best(d.top, d.at, d.top_z, s);
    if (tid == 0) { s.best = d.top; s.best_col = d.at; s.best_z = d.top_z; }
  }
  // The smallest z that min-p keeps: at most the largest of the row.
  __device__ __noinline__ float least_kept(float min_p) const {
    const double least = (double)zmax + log(fmin((double)min_p, 1.));
    float z = (float)least;
    if ((double)z < least) z = nextafterf(z, INFINITY);
    return fmaxf(z, -SF_MAX);
  }
  // What stands in the list of top-p for a logit: z where the order is not that of the logits.
  __device__ __forceinline__ float listed(float x) const { return sizeof(T) == 4 ? sf_quotient(x, temperature) : x; }
  // The first block: divides the list's entries, from which on what is compared is z.
  __device__ __noinline__ void divide_list(int n) {
    for (int i = tid; i < n; i += SF_THREADS) {
      const unsigned long long e = s.list[i];
      s.list[i] = (unsigned long long)(~sf_key(quotient(sf_entry_x(e)) + 0.f)) << 32 | (unsigned)e;
    }
    __syncthreads();
    to_z();
  }
  // The first block: top-k (0: none), then top-p of `goal`, or of the share top_p of what top-k kept, then the floor and the draw, in
  // a list of n <= SF_THREADS tokens that holds all that is kept.
  __device__ __noinline__ void finish_few(int n, int top_k, double top_p, double goal, float floor) {
    const Place p = place_of(s.list, n, top_k);
    const float x = sf_entry_x(p.entry);
    bool kept = p.valid;
    if (top_k > 0) {
      kept = kept && p.is_k;
      goal = top_p < 1. ? fmax(0., top_p * ((double)sf_block_count(kept ? p.own : 0, s) / SF_UNIT)) : INFINITY;
    }
    kept = kept && (p.rank == 0 || (double)p.before / SF_UNIT <= goal) && x >= floor;
    float best = -INFINITY, best_z = 0.f;
    int col = -1;
    if (kept) {
      const float z = quotient(x);
      sf_better(best, col, best_z, greedy ? z : z + noise(sf_bits(word, (unsigned)p.entry)), (int)(unsigned)p.entry, z);
    }
    const unsigned long long sum = sf_block_count(kept ? p.own : 0, s);
    sf_block_best(best, col, best_z, s);
    write(best_z, col, (double)sum / SF_UNIT);
  }
  // The first block, for top-p: its list of n tokens without those that are lighter than room / n, the mass that may be left out
  // parted among them.  `total`: the row's mass; returns how many are left.
  __device__ __noinline__ int thin_out(int n, double goal, double total) {
    constexpr int E = SF_LIST / SF_THREADS;
    unsigned long long e[E], sum = 0;
    float w[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const bool in = tid + i * SF_THREADS < n;
      e[i] = in ? s.list[tid + i * SF_THREADS] : ~0ull;
      w[i] = in ? weight(sf_entry_x(e[i])) : 0.f;
      sum += whole((double)w[i]);
    }
    if (tid == 0) s.list_n = 0;
    // what is not in the list is left out; a little more for the sums' rounding
    const double in_list = (double)sf_block_count(sum, s) / SF_UNIT, room = fmin(in_list, total) - goal - 2e-5 * total;
    const float least = (float)(fmax(room, 0.) / n * 0.999);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (tid + i * SF_THREADS < n && w[i] >= least) s.list[atomicAdd(&s.list_n, 1u)] = e[i];
    __syncthreads();
    return (int)s.list_n;
  }
  // The first block: top-k, then top-p, then the draw, in a list that holds the k largest.
  __device__ __noinline__ void top_k_of_list(int n, int top_k, bool by_p, float top_p, float floor) {
    if (n <= SF_THREADS) {
      finish_few(n, top_k, by_p ? (double)top_p : 1., 0., floor);
      return;
    }
    list_border(n, false, (double)top_k, 0, 0.);
    const float border = s.border;
    if (by_p) {
      // of the k-th and its equals, which move to the front
      __syncthreads();
      if (tid == 0) s.list_n = 0;
      constexpr int E = SF_LIST / SF_THREADS;
      unsigned long long e[E], w = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) e[i] = tid + i * SF_THREADS < n ? s.list[tid + i * SF_THREADS] : ~0ull;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (tid + i * SF_THREADS < n && sf_entry_x(e[i]) >= border) {
          w += whole((double)weight(sf_entry_x(e[i])));
          s.list[atomicAdd(&s.list_n, 1u)] = e[i];
        }
      const double mass = (double)sf_block_count(w, s) / SF_UNIT;
      n = (int)s.list_n;
      list_border(n, true, fmax(0., (double)top_p * mass), 0, 0.);
    }
    finish_list(n, s.border, s.border_col, floor);
  }

  __device__ __noinline__ void run() {
    const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;
    const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
    const bool by_k = top_k > 0 && top_k < a.V, by_p = top_p < 1.f;
    cluster.sync();  // what fast() has left may still be read
    if (divided) to_z();
    // ---- the maximum, and the mass relative to each thread's own ----
    float mine, part;
    for (;;) {
      mine = -INFINITY;
      part = 0.f;
      const SfRow<T> q = r;
      const float k = c;
      q.each([&](float x, int) {
        if (x > mine) {  // rare after the first few
          part *= exp2f((mine - x) * k);  // 0 at first: exp2(-inf)
          mine = x;
        }
        if (x >= -SF_MAX) part += exp2f((x - mine) * k);
      });
      float mx = warp_max(mine);
      if ((tid & 31) == 0) s.red[0][tid >> 5] = mx;
      __syncthreads();
      mx = (float)s.red[0][0];
      for (int w = 1; w < SF_WARPS; ++w) mx = fmaxf(mx, (float)s.red[0][w]);
      const double sum = sf_block_sum(mine == -INFINITY ? 0. : (double)(part * exp2f((mine - mx) * c)), s);
      if (tid == 0) {
        s.fmax = mx;
        s.first_mass = sum;
      }
      cluster.sync();
      xmax = max_of([](const SfShared& o) { return o.fmax; });
      if (divided || !(xmax > r.cap)) break;
      read_divided(true);  // 16-bit logits of which some have no finite quotient: once more, as z
      to_z();
      cluster.sync();
    }
    zmax = quotient(xmax);
    if (zmax == -INFINITY) {  // nothing to draw from
      if (rank == 0 && tid == 0) { a.tok[row] = 0; a.logp[row] = -INFINITY; }
      return;
    }
    const double total = sum_of([&](const SfShared& o) { return o.fmax > -INFINITY ? o.first_mass * (double)exp2f((o.fmax - xmax) * c) : 0.; });
    const float floor = min_p > 0.f ? least_of(least_kept(min_p)) : -INFINITY;
    float border = -INFINITY;
    int border_col = 0x7fffffff;
    double kept = 0.;
    if (by_k) {
      int n = 0;
      if (top_k <= C * SF_THREADS) {
        // the bin of the k-th largest of the threads' maxima: at least k tokens lie in it or above
        step = 64.f / temperature;
        clear_hist();
        if (mine > -INFINITY) atomicAdd(&s.hist[pass().linear_bin(mine)], 1u);
        unsigned h[SF_EACH];
        merged_bins(h);
        cluster.sync();
        if (tid == 0) s.bin_lo = SF_BINS;
        __syncthreads();
        bracket_count(h, (unsigned)top_k);
        const int last = s.bin_lo;
        __syncthreads();
        if (last < SF_BINS - 1) {
          const float from = fmaxf(-SF_MAX, xmax - (float)(last + 1) / step * 1.000001f);  // a little below the bin's end
          n = gather([&](float x) { return x >= from; });
        }
      }
      double goal = (double)top_k;
      if (n == 0) n = search(false, goal, false, -INFINITY, border, border_col, kept);
      if (n > 0) {
        if (rank == 0) top_k_of_list(n, top_k, by_p, top_p, floor);
        return;
      }
    }
    if (by_p) {
      int n = 0;
      double goal = fmax(0., (double)top_p * total);
      float from = border;
      if (by_k) {
        goal = fmax(0., (double)top_p);
      } else {
        // lighter tokens than this together have less than what top-p leaves out; a little is added for the sums' rounding
        const double least = (1. - (double)top_p - 2e-5) * total / a.V;
        if (least > 0.) from = fmaxf(-SF_MAX, xmax + ((float)log(least) - 1e-3f) * temperature);
        // weights are at most 1: at least `goal` tokens are kept, and with many of them come more than the list holds
        if (least > 0. && goal < SF_LIST / 16) n = gather([&](float x) { return x >= from; });
      }
      if (n == 0) n = search(true, goal, by_k, from, border, border_col, kept);
      if (n > 0) {
        if (rank == 0) {
          list_border(n, true, goal, 0, 0.);
          finish_list(n, s.border, s.border_col, floor);
        }
        return;
      }
    }
    const bool all = border == -INFINITY && floor == -INFINITY;  // then the mass is known
    if (floor > border) { border = floor; border_col = 0x7fffffff; kept = 0.; }
    // ---- what is kept: its mass, and the draw ----
    double mass = all ? total : kept;
    if (mass == 0.) {
      part = 0.f;
      const Pass q = pass();
      const float last = border;
      const int last_col = border_col;
      q.r.each([&](float x, int col) {
        if (within(x, col, last, last_col) && x >= -SF_MAX) part += q.weight(x);
      });
      mass = cluster_sum((double)part);
    }
    const double reached = (double)zmax + log(mass) - 3.;
    float best = -INFINITY, best_z = 0.f;
    int col = -1;
    for (int turn = 0; turn < 2 && (col < 0 || (!greedy && (double)best < reached)); ++turn) {
      const Pass q = pass();
      const float reach = turn == 1 ? INFINITY : (float)(20.0855369 * 1.001 / mass), last = fmaxf(border, -SF_MAX), t = temperature;
      const int last_col = border == -INFINITY ? 0x7fffffff : border_col;
      const uint32_t w = word;
      const bool most = greedy, as = as_sampler;
      float top = -INFINITY, top_z = 0.f;
      int at = -1;
      q.r.each([&](float x, int i) {
        if (within(x, i, last, last_col)) consider(x, i, q.weight(x), reach, t, w, most, as, top, at, top_z);
      });
      best = top;
      best_z = top_z;
      col = at;
      if (greedy && col >= 0) best_z = quotient(best_z);
      sf_block_best(best, col, best_z, s);
      if (tid == 0) { s.best = best; s.best_col = col; s.best_z = best_z; }
      cluster.sync();
      for (int b = 0; b < C; ++b) sf_better(best, col, best_z, of(b)->best, of(b)->best_col, of(b)->best_z);
      cluster.sync();
    }
    if (rank == 0) write(best_z, col, mass);
  }
};

constexpr size_t SF_HEAD = (sizeof(SfShared) + 15) / 16 * 16;
// vecs, HELD: vectors of a row in each block's shared memory.
template <typename T, bool HELD>
__global__ void __launch_bounds__(SF_THREADS, 2)
sample_filtered_kernel(const __grid_constant__ SampleArgs a, int vecs) {
  extern __shared__ __align__(16) unsigned char raw[];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / C;
  pdl_launch_dependents();
  pdl_wait();
  SfSampler<T> f{*reinterpret_cast<SfShared*>(raw), cluster, a};
  constexpr int N = 16 / sizeof(T);
  const int per = ((a.V + C - 1) / C + N - 1) / N * N;  // a multiple of a vector
  f.r.x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.row_stride;
  f.r.v0 = min(a.V / N * N, rank * per);
  f.r.v1 = rank == C - 1 ? a.V : min(a.V / N * N, (rank + 1) * per);
  f.r.vec = (reinterpret_cast<uintptr_t>(f.r.x) & 15) == 0;
  const float temp = a.temperature ? a.temperature[row] : a.temperature_all;
  f.temperature = temp < 1e-6f ? 1e-6f : temp;
  f.c = SF_LOG2E / f.temperature;
  f.r.cap = SF_MAX * fminf(f.temperature, 1.f);
  f.read_divided(sizeof(T) == 4 || !(f.temperature >= SF_LOW && f.temperature <= SF_HIGH));
  f.greedy = !(temp > 0.f);
  f.as_sampler = a.words == nullptr;
  f.word = a.words ? a.words[row] : a.seed ^ sf_hash((a.step_ptr ? (uint32_t)*a.step_ptr : 0u) * 0x9E3779B9U + (uint32_t)row);
  f.C = C;
  f.rank = rank;
  f.row = row;
  f.tid = threadIdx.x;
  f.lead = cluster.map_shared_rank(&f.s, 0);
  const bool done = f.template fast<HELD>(reinterpret_cast<uint4*>(raw + SF_HEAD), vecs);
  if (done) return;  // the others may have left already
  f.run();           // all blocks of a cluster take the same way
  cluster.sync();    // no block leaves while another may read its shared memory
}

template <typename T, bool HELD>
void sample_filtered_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int B, int C, int vecs, cudaStream_t st) {
  cfg.gridDim = dim3((unsigned)(B * C));
  cfg.blockDim = dim3(SF_THREADS);
  cfg.dynamicSmemBytes = SF_HEAD + (size_t)vecs * 16;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = trlb_host::pdl_enabled() ? 2 : 1;
}
template <typename T, bool HELD>
cudaError_t sample_filtered_ready() {
  return cudaFuncSetAttribute(sample_filtered_kernel<T, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              (int)(SF_HEAD + (HELD ? SF_HELD * 16 : 0)));
}
// Clusters of C blocks that find a place at once, asked for once: on 148 SMs 148 of 2, 71 of 4, 56 of 5, 33 of 8.
template <typename T, bool HELD>
int sample_filtered_places(int device, int C) {
  static int known[64][9] = {};  // a second thread that asks at once writes the same
  if (device < 64 && known[device][C] > 0) return known[device][C];
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  sample_filtered_config<T, HELD>(cfg, attr, 1, C, HELD ? SF_HELD : 0, nullptr);
  cfg.numAttrs = 1;
  int n = 0;
  if (sample_filtered_ready<T, HELD>() != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, sample_filtered_kernel<T, HELD>, &cfg) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    n = 1;
  }
  if (device < 64) known[device][C] = n;
  return n;
}
template <typename T, bool HELD>
int sample_filtered_launch(const SampleArgs& a, int B, int C, int vecs, cudaStream_t st) {
  const cudaError_t e = sample_filtered_ready<T, HELD>();
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  sample_filtered_config<T, HELD>(cfg, attr, B, C, vecs, st);
  return (int)cudaLaunchKernelEx(&cfg, sample_filtered_kernel<T, HELD>, a, vecs);
}
template <typename T>
int sample_filtered_pick(const SampleArgs& a, int B, cudaStream_t st) {
  // Blocks a row, up to the 8 of a portable cluster: enough to hold it in their shared memory, and as many more as all rows find a
  // place for at once.  More rows than that are not held: they get as many blocks as find a place, and at least two, so that a long
  // row (top-p of a flat one takes five times as long as top-k) has two SMs.  Measured with 256 rows of 128256 fp32 logits, flat and
  // with top-p 0.95: held 315 us, two blocks 181, one block 165; with parameters of all kinds: 181, 114, 146.  64 rows of 152064 bf16
  // logits: held 64 us, not held 66; 32 of them with 8 blocks each 48, with 5 55; 72 of them: held in two waves 71, not held 77.
  constexpr long long N = 16 / sizeof(T);
  int device = 0, C = 1;
  const cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return (int)e;
  while (C < 8 && C * N * SF_HELD < a.V) ++C;
  if (C * N * SF_HELD >= a.V && sample_filtered_places<T, true>(device, C) >= B) {
    while (C < 8 && sample_filtered_places<T, true>(device, C + 1) >= B) ++C;
    return sample_filtered_launch<T, true>(a, B, C, (int)(((a.V + C - 1) / C + N - 1) / N), st);
  }
  C = 8;
  while (C > 2 && sample_filtered_places<T, false>(device, C) < B) --C;
  return sample_filtered_launch<T, false>(a, B, C, 0, st);
}

}  // namespace trlb

using namespace trlb;

// dtype: 0 bf16, 1 fp16, 2 fp32.  Per-row parameters may be null, then the number for all rows holds.  words null: the random
// word of a row is made of seed, *step_ptr and the row, as trlb_sample makes it.
struct SampleCall {
  const void* logits;
  const float* temperature;
  const int* top_k;
  const float *top_p, *min_p;
  const uint32_t* words;
  const int* step_ptr;
  int* tok;
  float* logp;
  cudaStream_t stream;
  long long row_stride;
  int dtype, B, V, top_k_all, unused;
  uint32_t seed;
  float temperature_all, top_p_all, min_p_all;
};
TRLB_API int trlb_sample_filtered(const SampleCall* call) {
  const SampleCall c = *call;
  if (c.B == 0) return 0;
  if (c.V < 1 || c.B < 0 || c.B > (1 << 27)) return -1;
  SampleArgs a{c.logits, c.row_stride, c.V, c.temperature, c.top_p, c.min_p, c.top_k, c.temperature_all, c.top_p_all, c.min_p_all,
               c.top_k_all, c.words, c.seed, c.step_ptr, c.tok, c.logp};
  if (c.dtype == 0) return sample_filtered_pick<__nv_bfloat16>(a, c.B, c.stream);
  if (c.dtype == 1) return sample_filtered_pick<__half>(a, c.B, c.stream);
  if (c.dtype == 2) return sample_filtered_pick<float>(a, c.B, c.stream);
  return -2;
}
