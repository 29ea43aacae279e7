// Sampling with temperature, top-k, top-p and min-p from one random word per row.
//
//   z = logit / max(temperature, 1e-6); NaN counts as -inf, +inf as the largest finite value
//   top-k keeps z >= the k-th largest (equals of the k-th too); 0 keeps all
//   top-p keeps, most likely first and the lower column first among equals, each token before which at most
//         top_p of the mass of what top-k kept stands
//   min-p keeps z >= max z + log(min_p)
//   token = argmax over what is kept of z - log(-log u), u = (hash(word of the row, column) + 1/2) / 2^32; of z where
//   temperature is 0; its log-probability is that in the distribution over what is kept
//
// All filters are one border: the last token kept, in the order "larger z, then lower column".  A row is read by the blocks
// of a cluster.  What bounds it is the row's bytes, which stay in the second-level cache after the first pass, and the
// latency of the few exchanges between the blocks; so the border is found in as few passes as the row allows:
//   1. the maximum;
//   2. a histogram of max z - z in steps of 1/64 and the mass; from counts alone the bins bound the mass above each of them
//      from both sides, which brackets the border;
//   3. the tokens of the bracket (and of all bins above, where they are few) are listed and sorted by one block, which finds
//      the border exactly.  Where the list holds every kept token it draws the token, too;
//   4. otherwise a last pass over the row sums what is kept and draws.
// A bracket with too many tokens for the list is cut again by histograms over the keys' bits.
// Counts are integers and sums are taken in a fixed order, so results do not depend on timing.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace trlb {

constexpr int SF_THREADS = 1024, SF_WARPS = SF_THREADS / 32;
constexpr int SF_BINS = 2048;      // histogram bins; bin SF_BINS holds what lies further below
constexpr int SF_LIST = 4096;      // tokens that the list holds
constexpr float SF_STEP = 64.f;    // bins per unit of z
constexpr float SF_MAX = 3.4028234663852886e38f;

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
// -log(-log u): both halves of (0, 1) in the form that keeps their precision
__device__ __forceinline__ float sf_gumbel(uint32_t word, uint32_t col) {
  const uint32_t h = sf_hash(sf_hash(word ^ sf_hash(col * 0x85EBCA6BU + 0x165667B1U)) + col);
  float e;
  if (h & 0x80000000u) e = -log1pf(-((float)(~h) + 0.5f) * 2.3283064365386963e-10f);
  else e = -logf(((float)h + 0.5f) * 2.3283064365386963e-10f);
  return -logf(e);
}
// Orders floats as unsigned integers.
__device__ __forceinline__ uint32_t sf_key(float z) {
  const uint32_t u = __float_as_uint(z);
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

// NaN counts as -inf; + 0 makes one zero of both, so that their bits are equal, too
__device__ __forceinline__ float sf_z(float x, float T) {
  const float z = __fdiv_rn(x, T);
  return z != z ? -INFINITY : fminf(z, SF_MAX) + 0.f;
}

struct SfShared {
  unsigned hist[SF_BINS];
  unsigned long long list[SF_LIST];  // ~key << 32 | column: ascending is "larger z, then lower column"
  double red[3][SF_WARPS];
  double mass;                       // this block's share of a sum
  float fmax;
  unsigned kmin, kmax, list_n;
  int bin_lo, bin_hi;                // the bracket, its tokens and those above it: the same in every block
  unsigned above, upto;
  float border_z;                    // written by the first block, read by all
  int border_col;
  float best;                        // this block's draw
  int best_col;
  float best_z;
};

template <typename T>
struct SfRow {
  const T* x;
  int v0, v1;       // this block's columns
  bool vec;
  float temperature;
  // f(z, column) over the block's columns
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int N = 16 / sizeof(T);
    if (vec) {
      const int n0 = v0 / N, n1 = v1 / N;  // v0 is a multiple of N
      for (int i = n0 + threadIdx.x; i < n1; i += SF_THREADS) {
        float y[N];
        sf_unpack<T>(reinterpret_cast<const uint4*>(x)[i], y);
#pragma unroll
        for (int k = 0; k < N; ++k) f(sf_z(y[k], temperature), i * N + k);
      }
      for (int i = n1 * N + threadIdx.x; i < v1; i += SF_THREADS) f(sf_z(sf_load(x, i), temperature), i);
    } else {
      for (int i = v0 + threadIdx.x; i < v1; i += SF_THREADS) f(sf_z(sf_load(x, i), temperature), i);
    }
  }
};

__device__ __forceinline__ double sf_block_sum(double v, SfShared& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.red[0][threadIdx.x >> 5] = v;
  __syncthreads();
  double all = 0.;
  for (int w = 0; w < SF_WARPS; ++w) all += s.red[0][w];
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

// Sorts the first n entries of the list ascending (n <= SF_LIST).
__device__ void sf_sort(SfShared& s, int n) {
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += SF_THREADS) s.list[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += SF_THREADS) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const unsigned long long x = s.list[a], y = s.list[b];
        if ((x > y) == ((a & k) == 0)) { s.list[a] = y; s.list[b] = x; }
      }
      __syncthreads();
    }
}
__device__ __forceinline__ float sf_list_z(unsigned long long e) { return sf_unkey(~(unsigned)(e >> 32)); }

// Draw and log-probability from the blocks' (or threads') parts: the larger key, then the lower column.
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
    s.red[0][threadIdx.x >> 5] = best;
    s.red[1][threadIdx.x >> 5] = col;
    s.red[2][threadIdx.x >> 5] = z;
  }
  __syncthreads();
  for (int w = 0; w < SF_WARPS; ++w) sf_better(best, col, z, (float)s.red[0][w], (int)s.red[1][w], (float)s.red[2][w]);
}

template <typename T>
struct SfSampler {
  SfShared& s;
  cg::cluster_group cluster;
  const SampleArgs& a;
  SfRow<T> r;
  int C, rank, row, tid;
  float zmax;
  uint32_t word;
  bool greedy;
  SfShared* lead;

  __device__ __forceinline__ SfShared* of(int c) { return cluster.map_shared_rank(&s, c); }
  __device__ __forceinline__ float weight(float z) const { return expf(z - zmax); }
  __device__ __forceinline__ float key_of(float z, int col) const { return greedy ? z : z + sf_gumbel(word, (uint32_t)col); }
  __device__ __forceinline__ int linear_bin(float z) const { return (int)fminf((zmax - z) * SF_STEP, (float)(SF_BINS - 1)); }

  // Sum of a block-wide value over the cluster, in the order of the blocks.  Ends with a barrier.
  __device__ double cluster_sum(double v) {
    v = sf_block_sum(v, s);
    if (tid == 0) s.mass = v;
    cluster.sync();
    double all = 0.;
    for (int c = 0; c < C; ++c) all += of(c)->mass;
    cluster.sync();
    return all;
  }
  __device__ void clear_hist() {
    for (int i = tid; i < SF_BINS; i += SF_THREADS) s.hist[i] = 0;
    __syncthreads();
  }
  // This thread's two bins of the whole row.
  __device__ void merged_bins(unsigned (&n)[2]) {
    cluster.sync();
    n[0] = n[1] = 0;
    for (int c = 0; c < C; ++c) {
      n[0] += of(c)->hist[2 * tid];
      n[1] += of(c)->hist[2 * tid + 1];
    }
    cluster.sync();
  }
  // The bin of the k-th token of the histogram.
  __device__ void bracket_count(const unsigned (&n)[2], unsigned k) {
    double v[1] = {(double)n[0] + n[1]};
    sf_block_prefix(v, s);
    const unsigned upto = (unsigned)v[0], below = upto - n[0] - n[1];
    if (below < k && k <= upto) {
      const bool first = k <= below + n[0];
      s.bin_lo = s.bin_hi = 2 * tid + (first ? 0 : 1);
      s.above = below + (first ? 0 : n[0]);
      s.upto = below + n[0] + (first ? 0 : n[1]);
    }
    __syncthreads();
  }
  // Bins between which the mass passes `goal`: the first whose upper bound of the mass up to it does, to the first whose
  // lower bound does.  hi / lo: bounds of a token's weight in this thread's bins; mass: what stands above the histogram.
  __device__ void bracket_mass(const unsigned (&n)[2], const float (&hi)[2], const float (&lo)[2], double mass, double goal) {
    if (tid == 0) {
      s.bin_lo = s.bin_hi = SF_BINS - 1;
      s.above = s.upto = 0;
    }
    double v[3] = {(double)n[0] + n[1], (n[0] * (double)hi[0] + n[1] * (double)hi[1]) * 1.00001,
                   (n[0] * (double)lo[0] + n[1] * (double)lo[1]) * 0.99999};
    const double own_hi = v[1], own_lo = v[2];
    sf_block_prefix(v, s);
    const unsigned below = (unsigned)v[0] - n[0] - n[1];
    double up = mass + (v[1] - own_hi), low = mass + (v[2] - own_lo);  // bounds before this thread's bins
    unsigned cnt = below;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double up1 = up + n[i] * (double)hi[i] * 1.00001, low1 = low + n[i] * (double)lo[i] * 0.99999;
      if (up1 > goal) atomicMin(&s.bin_lo, 2 * tid + i);
      if (low1 > goal) atomicMin(&s.bin_hi, 2 * tid + i);
      up = up1;
      low = low1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (2 * tid + i == s.bin_lo) s.above = cnt;
      cnt += n[i];
      if (2 * tid + i == s.bin_hi) s.upto = cnt;
      s.hist[2 * tid + i] = cnt;  // from here on: tokens up to and with a bin
    }
    __syncthreads();
  }
  // Lists the row's tokens that `in` takes in the first block, sorted; returns their number (to all blocks).
  template <typename F>
  __device__ int gather(F in) {
    if (tid == 0) s.list_n = 0;
    __syncthreads();
    r.each([&](float z, int col) {
      if (in(z)) {
        const unsigned i = atomicAdd(&s.list_n, 1u);
        if (i < SF_LIST) s.list[i] = (unsigned long long)(~sf_key(z)) << 32 | (unsigned)col;
      }
    });
    cluster.sync();
    int n = 0;
    for (int c = 0; c < C; ++c) {
      const int m = min((int)of(c)->list_n, SF_LIST - n);
      if (rank == 0 && c > 0) {
        const unsigned long long* from = of(c)->list;
        for (int i = tid; i < m; i += SF_THREADS) s.list[n + i] = from[i];
      }
      n += m;
    }
    if (rank == 0) {
      __syncthreads();
      sf_sort(s, n);
    }
    return n;
  }
  // The sorted list's last entry before which at most `goal` of mass stands, `mass` of it above the list.
  __device__ int last_within(int n, double mass, double goal) {
    constexpr int E = SF_LIST / SF_THREADS;
    double v[1] = {0.}, w[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = tid * E + e;
      w[e] = i < n ? (double)weight(sf_list_z(s.list[i])) : 0.;
      v[0] += w[e];
    }
    const double own = v[0];
    sf_block_prefix(v, s);
    if (tid == 0) s.bin_lo = 0;
    __syncthreads();
    double before = mass + (v[0] - own);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = tid * E + e;
      if (i < n && before <= goal) atomicMax(&s.bin_lo, i);
      before += w[e];
    }
    __syncthreads();
    return s.bin_lo;
  }
  // Sums and draws over the first n list entries with z >= floor.  First block only.
  __device__ void finish_list(int n, float floor) {
    double mass = 0.;
    float best = -INFINITY, best_z = 0.f;
    int col = -1;
    for (int i = tid; i < n; i += SF_THREADS) {
      const unsigned long long e = s.list[i];
      const float z = sf_list_z(e);
      if (z < floor) continue;
      mass += (double)weight(z);
      sf_better(best, col, best_z, key_of(z, (int)(unsigned)e), (int)(unsigned)e, z);
    }
    mass = sf_block_sum(mass, s);
    sf_block_best(best, col, best_z, s);
    write(best_z, col, mass);
  }
  __device__ void write(float z, int col, double mass) {
    if (tid == 0) {
      a.tok[row] = col;
      a.logp[row] = (float)((double)z - (double)zmax - log(mass));
    }
  }

  // The border of top-k (by_mass false: goal is k) or top-p (goal is p) among the tokens with z >= floor.  Returns the number
  // of entries of the first block's list if that holds every token down to the border's bin, else 0 and the border.
  __device__ int search(bool by_mass, double goal, float floor, float& border_z, int& border_col, double& total) {
    clear_hist();
    float part = 0.f;
    r.each([&](float z, int) {
      if (z >= floor && z > -INFINITY) {
        atomicAdd(&s.hist[linear_bin(z)], 1u);
        part += weight(z);
      }
    });
    total = cluster_sum((double)part);
    unsigned n[2];
    merged_bins(n);
    double limit = 0.;
    if (by_mass) {
      limit = fmax(0., goal * total);
      float hi[2], lo[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int bin = 2 * tid + i;
        hi[i] = expf(-(float)bin / SF_STEP);
        lo[i] = bin == SF_BINS - 1 ? 0.f : expf(-(float)(bin + 1) / SF_STEP);
      }
      bracket_mass(n, hi, lo, 0., limit);
    } else {
      double all[1] = {(double)n[0] + n[1]};
      sf_block_prefix(all, s);
      if (tid == SF_THREADS - 1) s.upto = (unsigned)all[0];
      __syncthreads();
      const unsigned finite = s.upto;
      __syncthreads();
      if (goal > (double)finite) {  // fewer tokens than k: all are kept
        border_z = -INFINITY;
        border_col = 0x7fffffff;
        return 0;
      }
      bracket_count(n, (unsigned)goal);
    }
    const int b0 = s.bin_lo, b1 = s.bin_hi;
    unsigned above = s.above, upto = s.upto;
    __syncthreads();
    if (upto <= SF_LIST)
      return gather([&](float z) { return z >= floor && z > -INFINITY && linear_bin(z) <= b1; });
    auto member = [&](float z) {
      if (!(z >= floor && z > -INFINITY)) return false;
      const int b = linear_bin(z);
      return b >= b0 && b <= b1;
    };
    // keys of the bracket, and the mass above it
    unsigned kmin = 0xffffffffu, kmax = 0u;
    part = 0.f;
    r.each([&](float z, int) {
      if (member(z)) {
        kmin = min(kmin, sf_key(z));
        kmax = max(kmax, sf_key(z));
      } else if (z > -INFINITY && linear_bin(z) < b0) {
        part += weight(z);
      }
    });
    kmin = __reduce_min_sync(0xffffffffu, kmin);
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if (tid == 0) { s.kmin = 0xffffffffu; s.kmax = 0u; }
    __syncthreads();
    if ((tid & 31) == 0) { atomicMin(&s.kmin, kmin); atomicMax(&s.kmax, kmax); }
    double mass = cluster_sum((double)part);  // its barriers show kmin and kmax, too
    for (int c = 0; c < C; ++c) {
      kmin = min(kmin, of(c)->kmin);
      kmax = max(kmax, of(c)->kmax);
    }
    cluster.sync();
    // all tokens with keys in [kmin, kmax] are the bracket's: the bins are intervals of z.  Each turn leaves an interval of
    // one bin's width, so there are three at most.
    while (upto - above > SF_LIST && kmin < kmax) {
      int shift = 0;
      while (((kmax - kmin) >> shift) >= SF_BINS) ++shift;
      const unsigned top = kmax, span = kmax - kmin;
      clear_hist();
      r.each([&](float z, int) {
        const unsigned k = sf_key(z);
        if (k >= kmin && k <= top) atomicAdd(&s.hist[(top - k) >> shift], 1u);
      });
      merged_bins(n);
      unsigned c0, c1, a0, a1;  // the bracket's bins; tokens of the interval above it, and up to its end
      if (by_mass) {
        float hi[2], lo[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const unsigned bin = (unsigned)(2 * tid + i);
          hi[i] = lo[i] = 0.f;
          if (bin <= span >> shift) {
            hi[i] = weight(sf_unkey(top - (bin << shift)));
            const unsigned down = (bin << shift) + ((1u << shift) - 1u);
            lo[i] = weight(sf_unkey(top - min(down, span)));
          }
        }
        bracket_mass(n, hi, lo, mass, limit);
        c0 = (unsigned)s.bin_lo, c1 = (unsigned)s.bin_hi, a0 = s.above, a1 = s.upto;
        __syncthreads();
        auto between = [&](unsigned from, unsigned to) {  // exact mass of a run of bins
          float sum = 0.f;
          r.each([&](float z, int) {
            const unsigned k = sf_key(z);
            if (k >= kmin && k <= top && (top - k) >> shift >= from && (top - k) >> shift <= to) sum += weight(z);
          });
          return cluster_sum((double)sum);
        };
        if (c0 > 0) mass += between(0, c0 - 1);
        // the bounds leave several bins only where the goal is within their margin of a bin's end
        while (c0 < c1 && a1 - a0 > SF_LIST) {
          const unsigned mid = (c0 + c1) / 2, am = s.hist[mid];
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
      const int m = gather([&](float z) { const unsigned k = sf_key(z); return k >= kmin && k <= kmax; });
      if (rank == 0) {
        int at;
        if (by_mass) at = last_within(m, mass, limit);
        else at = (int)((unsigned)goal - above) - 1;
        if (tid == 0) {
          s.border_z = sf_list_z(s.list[at]);
          s.border_col = by_mass ? (int)(unsigned)s.list[at] : 0x7fffffff;
        }
      }
      cluster.sync();
      border_z = lead->border_z;
      border_col = lead->border_col;
      cluster.sync();
      return 0;
    }
    // more equals than the list holds
    border_z = sf_unkey(kmax);
    border_col = 0x7fffffff;
    if (by_mass) {
      const double w = (double)weight(border_z), equals = (double)(upto - above);
      const double fit = w > 0. ? ::floor((limit - mass) / w) + 1. : equals;  // how many of them are kept
      if (fit < equals) border_col = column_of(kmax, (unsigned)fmax(1., fit));
    }
    return 0;
  }
  // The column of the n-th token (in the order of the columns, from 1) whose key is `key`.
  __device__ int column_of(unsigned key, unsigned n) {
    int width = (a.V + SF_BINS - 1) / SF_BINS;
    clear_hist();
    r.each([&](float z, int col) { if (sf_key(z) == key) atomicAdd(&s.hist[col / width], 1u); });
    unsigned m[2];
    merged_bins(m);
    bracket_count(m, n);
    const int bin = s.bin_lo;
    const unsigned before = s.above;
    __syncthreads();
    if (rank == 0 && tid == 0) {  // some hundred columns: one thread counts its way through them
      const int lo = bin * width, hi = min(a.V, lo + width);
      unsigned count = before;
      int found = hi - 1;
      for (int c = lo; c < hi; ++c)
        if (sf_key(sf_z(sf_load(r.x, c), r.temperature)) == key && ++count == n) { found = c; break; }
      s.border_col = found;
    }
    cluster.sync();
    const int col = lead->border_col;
    cluster.sync();
    return col;
  }

  __device__ void run() {
    const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all;
    const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
    const bool by_k = top_k > 0 && top_k < a.V, by_p = top_p < 1.f;
    float mx = -INFINITY;
    r.each([&](float z, int) { mx = fmaxf(mx, z); });
    mx = warp_max(mx);
    if ((tid & 31) == 0) s.red[0][tid >> 5] = mx;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < SF_WARPS; ++w) mx = fmaxf(mx, (float)s.red[0][w]);
      s.fmax = mx;
    }
    cluster.sync();
    zmax = -INFINITY;
    for (int c = 0; c < C; ++c) zmax = fmaxf(zmax, of(c)->fmax);
    if (zmax == -INFINITY) {  // nothing to draw from
      if (rank == 0 && tid == 0) { a.tok[row] = 0; a.logp[row] = -INFINITY; }
      return;
    }
    float floor = -INFINITY;  // min-p, as the smallest value that it keeps
    if (min_p > 0.f) floor = fminf(zmax, __double2float_ru((double)zmax + log((double)min_p)));
    float bz = -INFINITY;
    int bc = 0x7fffffff;
    double total = 0.;
    if (by_k) {
      const int n = search(false, (double)top_k, -INFINITY, bz, bc, total);
      if (n > 0) {
        if (rank == 0) {
          const float zk = sf_list_z(s.list[top_k - 1]);
          double count = 0.;  // the k-th and its equals
          for (int i = tid; i < n; i += SF_THREADS) count += sf_list_z(s.list[i]) >= zk;
          int kept = (int)sf_block_sum(count, s);
          if (by_p) {
            double mass = 0.;
            for (int i = tid; i < kept; i += SF_THREADS) mass += (double)weight(sf_list_z(s.list[i]));
            mass = sf_block_sum(mass, s);
            kept = last_within(kept, 0., fmax(0., (double)top_p * mass)) + 1;
          }
          finish_list(kept, floor);
        }
        return;
      }
    }
    if (by_p) {
      const int n = search(true, (double)top_p, bz, bz, bc, total);
      if (n > 0) {
        if (rank == 0) finish_list(last_within(n, 0., fmax(0., (double)top_p * total)) + 1, floor);
        return;
      }
    }
    if (floor > bz) { bz = floor; bc = 0x7fffffff; }
    float part = 0.f, best = -INFINITY, best_z = 0.f;
    int col = -1;
    r.each([&](float z, int c) {
      if (z == -INFINITY || z < bz || (z == bz && c > bc)) return;
      part += weight(z);
      const float k = key_of(z, c);
      if (col < 0 || k > best || (k == best && c < col)) { best = k; col = c; best_z = z; }
    });
    const double mass = cluster_sum((double)part);
    sf_block_best(best, col, best_z, s);
    if (tid == 0) { s.best = best; s.best_col = col; s.best_z = best_z; }
    cluster.sync();
    if (rank == 0) {
      for (int c = 1; c < C; ++c) sf_better(best, col, best_z, of(c)->best, of(c)->best_col, of(c)->best_z);
      write(best_z, col, mass);
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(SF_THREADS, 1)
sample_filtered_kernel(const __grid_constant__ SampleArgs a) {
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
  f.r.temperature = fmaxf(temp, 1e-6f);
  f.greedy = !(temp > 0.f);
  f.word = a.words ? a.words[row] : a.seed ^ sf_hash((a.step_ptr ? (uint32_t)*a.step_ptr : 0u) * 0x9E3779B9U + (uint32_t)row);
  f.C = C;
  f.rank = rank;
  f.row = row;
  f.tid = threadIdx.x;
  f.lead = cluster.map_shared_rank(&f.s, 0);
  f.run();
  cluster.sync();  // no block leaves while another may read its shared memory
}

template <typename T>
int sample_filtered_launch(const SampleArgs& a, int B, cudaStream_t st) {
  // blocks a row: as many as give every SM one, up to the 8 of a portable cluster
  int C = 1;
  while (C < 8 && 2 * C * B <= trlb_host::sm_count()) C *= 2;
  const size_t smem = sizeof(SfShared);
  cudaError_t e = cudaFuncSetAttribute(sample_filtered_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * C));
  cfg.blockDim = dim3(SF_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = trlb_host::pdl_enabled() ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, sample_filtered_kernel<T>, a);
}

}  // namespace trlb

using namespace trlb;

// dtype: 0 bf16, 1 fp16, 2 fp32.  Per-row parameters may be null, then the scalar beside them holds for every row.
// words null: the random word of a row is made of seed, *step_ptr and the row, as trlb_sample makes it.
TRLB_API int trlb_sample_filtered(const void* logits, int dtype, long long row_stride, int B, int V, const float* temperature,
                                  float temperature_all, const int* top_k, int top_k_all, const float* top_p, float top_p_all,
                                  const float* min_p, float min_p_all, const unsigned* words, unsigned seed,
                                  const int* step_ptr, int* tok, float* logp, cudaStream_t st) {
  if (B == 0) return 0;
  if (V < 1 || B < 0 || B > (1 << 27)) return -1;
  SampleArgs a{logits, row_stride, V, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, words,
               seed, step_ptr, tok, logp};
  if (dtype == 0) return sample_filtered_launch<__nv_bfloat16>(a, B, st);
  if (dtype == 1) return sample_filtered_launch<__half>(a, B, st);
  if (dtype == 2) return sample_filtered_launch<float>(a, B, st);
  return -2;
}
