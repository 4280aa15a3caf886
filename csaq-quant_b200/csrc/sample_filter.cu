// Sampling under temperature, top-k, top-p and min-p from given random numbers.
//
// Row m, with w_j = exp((x_j - max x) / T) and tokens ranked by falling logit,
// the lower index first among equals:
//   top-k  keeps the first k ranks,
//   top-p  of those the ranks whose preceding mass is at most p times their sum,
//   min-p  of those the tokens with w_j >= min_p,
// and the token is the first index whose cumulative kept weight (index order)
// exceeds u times the kept mass. NaN and -inf logits are never drawn; a row of
// nothing else gives -1. A temperature that is not above 0 takes the first rank.
//
// The answer is an index, so there is no tolerance to hide in: a vocabulary of
// 128k has borders everywhere in [0, 1), and weights or sums in 32 bits would move
// some of them across u. Weights and sums are therefore fp64 (B200 runs it at half
// the fp32 rate), and no sum goes through an atomic: every order is fixed.
//
// A cluster of CTAs takes one row and keeps it in shared memory as ordered integer
// keys: one pass over the logits. What follows depends on the row's settings:
//
//  list    top-k up to kListK: a histogram of counts over bins of 1/32 nat below the
//          largest logit says which bins hold the first k ranks; their tokens, little
//          more than k, are gathered in one CTA, sorted, cut and drawn from there.
//  nucleus top-p alone: a histogram of (approximate) masses says near which bin the cut
//          lies; the exact mass above three bins and the sorted tokens of the three
//          give the cut, and a last pass over the row draws under it.
//  digits  anything else that cuts, and what the two above hand over (more tokens than
//          the list holds, a cut out of the bins' range): the cut is found three key
//          bits at a time; every thread adds its elements into 8 bins of its own, the
//          bins are summed in a fixed order over threads and CTAs, and the next pass
//          looks only at the bin that holds the cut.
//  none    no top-k, no top-p: the last pass alone.
//
// The histograms go through integer atomics and only say where to look; the answer
// never depends on them.

#include <atomic>

#include "common.cuh"

namespace csaq {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 8, kDigit = 3;  // of the digit passes; two warps sum a bin
constexpr int kHist = 1024;           // bins of 1 / kPerNat below the largest logit
constexpr float kPerNat = 32.0f;
constexpr int kList = 2048;           // tokens that are sorted at most
constexpr int kListK = 1024;          // ranks that a list may keep
constexpr int kMaxCluster = 8;
constexpr int kTable = 256;           // 2^(j / 256)
constexpr double kNegligible = -50.0;  // exp below this is taken as 0: 2e-22 of the largest weight
static_assert(kBins * 2 == kWarps && kList == 4 * kThreads && kHist == 2 * kThreads, "shares of a thread");

struct FilterArgs {
  const void* logits;
  int n_parts;
  int64_t part_stride, ld, part_len, V;
  csaq_sample_params p;
  const float* random;
  int64_t* out;
  int chunk;  // elements of a CTA's slice
};

// Keys order like the logits; 0 stands for NaN and -inf. -0 and +0 are one value.
template <typename T> struct KeyOf;
template <> struct KeyOf<float> {
  using K = uint32_t;
  static __device__ __forceinline__ K key(float x) {
    if (x != x || x == -INFINITY) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  }
};
template <typename T>
struct KeyOf16 {
  using K = uint16_t;
  static __device__ __forceinline__ K key(T v) {
    const float x = to_f32<T>(v);
    if (x != x || x == -INFINITY) return 0;
    const uint32_t b = x == 0.0f ? 0u : bits_of<T>(v);
    return (K)(b & 0x8000u ? ~b : b | 0x8000u);
  }
};
template <> struct KeyOf<__half> : KeyOf16<__half> {
  static __device__ __forceinline__ float value(uint32_t k) {
    return __half2float(__ushort_as_half((unsigned short)(k & 0x8000u ? k & 0x7fffu : ~k)));
  }
};
template <> struct KeyOf<__nv_bfloat16> : KeyOf16<__nv_bfloat16> {
  static __device__ __forceinline__ float value(uint32_t k) {
    return __bfloat162float(__ushort_as_bfloat16((unsigned short)(k & 0x8000u ? k & 0x7fffu : ~k)));
  }
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(r)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  return r;
}
__device__ __forceinline__ double remote_f64(const double* p, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t remote_u64(const uint64_t* p, uint32_t rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t remote_u32(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}

// a float's value as a double, by bits (subnormals come out near 2^-127, which next to
// another logit is all the same)
__device__ __forceinline__ double widen(float x) {
  const uint32_t b = __float_as_uint(x);
  return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));
}

// exp(d / T) for d / T in [kNegligible, 0], c = 256 / (T ln 2), it = 1 / T: table-driven
// reduction (Tang 1989): d / T = n ln2 / 256 + r, exp = 2^(n / 256) (1 + r + .. + r^4 / 24),
// |r| <= 0.00136: within 4e-15 of it
__device__ __forceinline__ double exp_tab(double d, double c, double it, const double* tab) {
  const double magic = 6755399441055744.0;  // 1.5 2^52: the sum's low word is the rounded integer
  const double t = fma(d, c, magic);
  const int n = __double2loint(t);
  const double r = fma(t - magic, -0.0027076061740622863, d * it);  // ln 2 / 256
  double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  p *= tab[n & (kTable - 1)];
  return __hiloint2double(__double2hiint(p) + ((n >> 8) << 20), __double2loint(p));
}

// Static shared memory; what other CTAs read is marked.
struct Shared {
  double tab[kTable];
  double red[2][kBins];  // read by others: this CTA's bin sums, alternating from pass to pass
  double tot[kBins];     // the row's
  double half[kWarps];
  double scan[kWarps];
  uint32_t iscan[kWarps];
  double x_mass;     // read by others
  double x_above;    // read by others
  uint32_t x_ties;   // read by others
  uint32_t x_max;    // read by others
  uint32_t x_count;  // read by others: tokens in this CTA's list
  uint32_t x_key, x_keep;  // read by others (CTA 0): the cut of a nucleus; x_keep 0: none was found
  uint32_t wmax[kWarps];
  int pick;
  uint32_t at;
  uint32_t hist[kHist];  // read by others
};

// exclusive prefix sums of N doubles a thread in thread order; the total
template <int N>
__device__ __forceinline__ double block_scan(const double (&v)[N], double (&before)[N], double* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double mine = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) mine += v[i];
  double incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  double wb = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) wb += warp_sums[w];
    all += warp_sums[w];
  }
  double x = __shfl_up_sync(0xffffffffu, incl, 1);
  x = wb + (lane == 0 ? 0.0 : x);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    before[i] = x;
    x += v[i];
  }
  return all;
}
__device__ __forceinline__ double block_sum(double v, double* warp_sums) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = v;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all += warp_sums[w];
  return all;
}

// bitonic sort of n (a power of two, at most kList) in shared memory, largest first
__device__ __forceinline__ void sort_down(uint64_t* v, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int a = 2 * i - (i & (step - 1)), b = a + step;
        const uint64_t x = v[a], y = v[b];
        if ((x < y) == ((a & size) == 0)) v[a] = y, v[b] = x;
      }
    }
  __syncthreads();
}
__device__ __forceinline__ int pow2_from(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

template <typename T>
struct Row {
  using KO = KeyOf<T>;
  using K = typename KO::K;
  const K* keys;  // the slice, in index order
  int n;
  int64_t first;  // index of its first element
  Shared* sh;
  uint8_t* work;  // kWorkBytes: the bins of the digit passes, or the list
  uint32_t rank, nc;
  int parity;
  bool top_inf;  // the largest logit is +inf: its like have weight 1, all else 0
  double xmax, inv_t, scale_t, lowest;
  float fmax, per_bin;
  uint32_t kmax;

  __device__ __forceinline__ double weight(uint32_t k) const {
    if (top_inf) return k == kmax ? 1.0 : 0.0;
    const double d = widen(KO::value(k)) - xmax;
    return d >= lowest ? exp_tab(d, scale_t, inv_t, sh->tab) : 0.0;
  }
  // bins below the largest logit, in exact order of the keys; kHist and more: none
  __device__ __forceinline__ float depth(uint32_t k) const { return (fmax - KO::value(k)) * per_bin; }

  // f(key) over the slice, and f(key, position)
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int PER = 16 / (int)sizeof(K);
    const int whole = n / PER;
    for (int i = threadIdx.x; i < whole; i += kThreads) {
      const uint4 u = reinterpret_cast<const uint4*>(keys)[i];
      const K* e = reinterpret_cast<const K*>(&u);
#pragma unroll
      for (int j = 0; j < PER; ++j) f((uint32_t)e[j], i * PER + j);
    }
    for (int i = whole * PER + threadIdx.x; i < n; i += kThreads) f((uint32_t)keys[i], i);
  }

  struct Cut {
    uint32_t key;   // lowest kept key
    double base;    // weight ranked above it
    double mass;    // weight at it
    double target;  // the bound that the weight ranked above a kept element meets
  };

  // The lowest-ranked element whose weight ranked above is at most the target, among
  // keys in [klo, kmax]; keys of `alone` count once, with weight `alone_w` (nothing
  // when 0). COUNT: weights 1 and target `bound`; else masses and target bound * total.
  template <bool COUNT>
  __device__ Cut select(uint32_t klo, double bound, uint32_t alone, double alone_w) {
    double* hist = reinterpret_cast<double*>(work);  // [bin][thread]
    const uint32_t span = kmax - klo;
    const int bits = 32 - __clz(span | 1u);
    uint32_t prefix = 0;
    Cut c{klo, 0.0, 0.0, bound};
    bool first_pass = true;
    __syncthreads();
    for (int shift = (bits - 1) / kDigit * kDigit; shift >= 0; shift -= kDigit) {
#pragma unroll
      for (int b = 0; b < kBins; ++b) hist[b * kThreads + threadIdx.x] = 0.0;
      each([&](uint32_t k, int) {
        const uint32_t o = k - klo;  // keys below klo wrap around to far above the span
        if (o > span || k == alone || (!first_pass && (o >> (shift + kDigit)) != prefix)) return;
        hist[((o >> shift) & (kBins - 1)) * kThreads + threadIdx.x] += COUNT ? 1.0 : weight(k);
      });
      if (alone_w != 0.0 && rank == 0 && threadIdx.x == 0) {
        const uint32_t o = alone - klo;
        if (o <= span && (first_pass || (o >> (shift + kDigit)) == prefix))
          hist[((o >> shift) & (kBins - 1)) * kThreads] += alone_w;
      }
      __syncthreads();
      {
        const int w = threadIdx.x >> 5, b = w >> 1, lane = threadIdx.x & 31;
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < kThreads / 64; ++i) s += hist[b * kThreads + (w & 1) * (kThreads / 2) + i * 32 + lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) sh->half[w] = s;
      }
      __syncthreads();
      if (threadIdx.x < kBins) sh->red[parity][threadIdx.x] = sh->half[2 * threadIdx.x] + sh->half[2 * threadIdx.x + 1];
      cluster_sync();
      if (threadIdx.x < kBins) {
        double s = 0.0;
        for (uint32_t r = 0; r < nc; ++r) s += remote_f64(&sh->red[parity][threadIdx.x], r);
        sh->tot[threadIdx.x] = s;
      }
      __syncthreads();
      parity ^= 1;
      if (first_pass && !COUNT) {
        double z = 0.0;
        for (int b = kBins - 1; b >= 0; --b) z += sh->tot[b];
        c.target = bound * z;
      }
      double above = c.base;
      int pick = 0;
      for (int b = kBins - 1; b >= 0; --b) {
        const double s = sh->tot[b];
        if (s > 0.0 && above <= c.target) pick = b, c.base = above, c.mass = s;
        above += s;
      }
      prefix = (prefix << kDigit) | (uint32_t)pick;
      first_pass = false;
      __syncthreads();  // tot is rewritten by the next pass
    }
    c.key = klo + prefix;
    return c;
  }

  // This CTA's histogram: counts, or masses as 2^15 w / 2^-bin (bin in units of 1 /
  // kPerNat nat); for masses the exact sum of the slice's weights comes back.
  template <bool COUNT>
  __device__ double histogram() {
    for (int i = threadIdx.x; i < kHist; i += kThreads) sh->hist[i] = 0;
    __syncthreads();
    double z = 0.0;
    each([&](uint32_t k, int) {
      if (k == 0) return;
      const float u = depth(k);
      if (!COUNT) z += weight(k);
      if (u < (float)kHist) {
        const int b = (int)u;
        atomicAdd(&sh->hist[b], COUNT ? 1u : (uint32_t)(32768.0f * __expf(((float)b - u) * (1.0f / kPerNat))));
      }
    });
    return COUNT ? 0.0 : block_sum(z, sh->scan);
  }
  // The row's histogram, bins 2 t and 2 t + 1 of thread t (after a cluster_sync).
  __device__ __forceinline__ void row_bins(double (&v)[2]) const {
    v[0] = v[1] = 0.0;
    for (uint32_t r = 0; r < nc; ++r) {
      v[0] += (double)remote_u32(&sh->hist[2 * threadIdx.x], r);
      v[1] += (double)remote_u32(&sh->hist[2 * threadIdx.x + 1], r);
    }
  }
  // The elements with lo <= depth < hi into this CTA's list; sh->x_count of them, or more than it holds.
  __device__ void gather(float lo, float hi) {
    uint64_t* list = reinterpret_cast<uint64_t*>(work);
    if (threadIdx.x == 0) sh->x_count = 0;
    __syncthreads();
    each([&](uint32_t k, int i) {
      if (k == 0) return;
      const float u = depth(k);
      if (u >= lo && u < hi) {
        const uint32_t at = atomicAdd(&sh->x_count, 1u);
        if (at < (uint32_t)kList) list[at] = (uint64_t)k << 32 | (0xffffffffu - (uint32_t)(first + i));
      }
    });
  }
  // CTA 0: all lists, sorted by rank (after a cluster_sync); the others are done with
  // theirs at the next one. -1: too many.
  __device__ int collect() {
    uint64_t* list = reinterpret_cast<uint64_t*>(work);
    uint32_t total = sh->x_count;
    for (uint32_t r = 1; r < nc; ++r) {
      const uint32_t c = remote_u32(&sh->x_count, r);
      if (total + c <= (uint32_t)kList)
        for (uint32_t i = threadIdx.x; i < c; i += kThreads) list[total + i] = remote_u64(list + i, r);
      total += c;
    }
    if (total > (uint32_t)kList) return -1;
    const int size = pow2_from((int)total);
    for (int i = (int)total + threadIdx.x; i < size; i += kThreads) list[i] = 0;
    sort_down(list, size);
    return (int)total;
  }
};
constexpr int kWorkBytes = kBins * kThreads * 8 > kList * 8 * 2 ? kBins * kThreads * 8 : kList * 8 * 2;

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_filter_kernel(const FilterArgs a) {
  using KO = KeyOf<T>;
  using K = typename KO::K;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Shared sh;
  pdl_wait();
  pdl_trigger();
  const uint32_t rank = cluster_rank(), nc = cluster_size();
  const int64_t m = blockIdx.x / nc;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  K* keys = reinterpret_cast<K*>(dyn + kWorkBytes);
  const int64_t lo = (int64_t)rank * a.chunk;
  const int n = (int)(lo >= a.V ? 0 : (a.V - lo < a.chunk ? a.V - lo : a.chunk));
  if (tid < kTable) sh.tab[tid] = exp2((double)tid / kTable);
  if (tid == 0) sh.pick = kThreads;

  // the slice as keys, and the largest of them
  uint32_t kmax = 0;
  constexpr int VE = 16 / (int)sizeof(T);
  const T* base = reinterpret_cast<const T*>(a.logits) + m * a.ld;
  const bool vec = reinterpret_cast<uintptr_t>(base) % 16 == 0 && a.part_len % VE == 0 && a.part_stride % VE == 0;
  int done = 0;
  if (vec) {
    for (int i = tid * VE; i + VE <= n; i += kThreads * VE) {
      const int64_t j = lo + i;
      const int64_t r = a.n_parts == 1 ? 0 : j / a.part_len;
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(base + r * a.part_stride + (j - r * a.part_len)));
      const T* e = reinterpret_cast<const T*>(&u);
      uint4 ku;
      K* ke = reinterpret_cast<K*>(&ku);
#pragma unroll
      for (int t = 0; t < VE; ++t) {
        ke[t] = KO::key(e[t]);
        kmax = max(kmax, (uint32_t)ke[t]);
      }
      *reinterpret_cast<uint4*>(keys + i) = ku;
    }
    done = n / VE * VE;
  }
  for (int i = done + tid; i < n; i += kThreads) {
    const int64_t j = lo + i;
    const int64_t r = a.n_parts == 1 ? 0 : j / a.part_len;
    const K k = KO::key(base[r * a.part_stride + (j - r * a.part_len)]);
    keys[i] = k;
    kmax = max(kmax, (uint32_t)k);
  }
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  if (lane == 0) sh.wmax[warp] = kmax;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 32; ++w) kmax = max(kmax, sh.wmax[w]);
    sh.x_max = kmax;
  }
  cluster_sync();
  kmax = 0;
  for (uint32_t r = 0; r < nc; ++r) kmax = max(kmax, remote_u32(&sh.x_max, r));

  if (kmax == 0) {  // nothing to draw, for every CTA of the row
    if (rank == 0 && tid == 0) a.out[m] = -1;
    cluster_sync();  // no CTA leaves while another reads its shared memory
    return;
  }
  const float temp = a.p.temperature ? a.p.temperature[m] : a.p.temperature_all;
  int top_k = a.p.top_k ? a.p.top_k[m] : a.p.top_k_all;
  const float top_p = a.p.top_p ? a.p.top_p[m] : a.p.top_p_all;
  double min_p = a.p.min_p ? a.p.min_p[m] : a.p.min_p_all;
  double u = a.random[m];
  const bool greedy = !(temp > 0.0f);
  if (greedy) top_k = 1;
  if (!(min_p > 0.0)) min_p = 0.0;
  if (min_p > 1.0) min_p = 1.0;
  if (!(u > 0.0)) u = 0.0;
  if (u >= 1.0) u = 1.0 - 0x1p-53;

  Row<T> row;
  row.keys = keys, row.n = n, row.first = lo, row.sh = &sh, row.work = dyn, row.rank = rank, row.nc = nc, row.parity = 0;
  row.kmax = kmax;
  const float xmax = KO::value(kmax);
  row.top_inf = xmax == INFINITY;
  row.xmax = widen(xmax);
  row.inv_t = greedy ? 1.0 : 1.0 / (double)temp;
  row.scale_t = row.inv_t * (kTable / 0.6931471805599453);
  row.lowest = kNegligible / row.inv_t;
  row.fmax = xmax;
  row.per_bin = fminf((float)(row.inv_t * kPerNat), 1e30f);

  // the lowest key that can have weight: a little below max + kNegligible T
  uint32_t klo = kmax;
  if (!row.top_inf) {
    const double x = row.xmax + (kNegligible - 1.0) / row.inv_t;
    klo = x > -3.0e38 ? KO::key(from_f32<T>((float)(x - fabs(x) * 0x1p-6))) : 1u;
    if (klo == 0 || klo > kmax) klo = 1u;
  }

  const bool cut_k = top_k > 0 && top_k < a.V, cut_p = top_p < 1.0f && !greedy;  // a NaN top_p switches it off
  const double p = top_p > 0.0f ? (double)top_p : 0.0;
  // keys above ckey are kept, and the first cties of those at it
  uint32_t ckey = klo, cties = 0xffffffffu;
  bool digits = cut_k || cut_p;
  // where differences of logits and their bins cannot overflow into one another
  const bool binned = fabsf(xmax) <= 1e38f && (greedy || temp <= 1e30f);

  if (cut_k && top_k <= kListK && binned) {
    row.template histogram<true>();
    cluster_sync();
    double v[2], before[2];
    row.row_bins(v);
    if (tid == 0) sh.at = kHist;
    block_scan<2>(v, before, sh.scan);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)  // the bin that the k-th rank falls into
      if (before[i] < (double)top_k && before[i] + v[i] >= (double)top_k) sh.at = 2 * tid + i;
    __syncthreads();
    const uint32_t at = sh.at;
    if (at < kHist) {
      row.gather(0.0f, (float)(at + 1));
      cluster_sync();
      uint32_t total = 0;
      for (uint32_t r = 0; r < nc; ++r) total += remote_u32(&sh.x_count, r);
      if (total <= (uint32_t)kList) {
        if (rank == 0) {
          uint64_t* list = reinterpret_cast<uint64_t*>(dyn);
          const int m1 = min(row.collect(), top_k);  // ranks 0 .. m1 - 1 pass top-k
          double w[2], above[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) w[i] = 2 * tid + i < m1 ? row.weight((uint32_t)(list[2 * tid + i] >> 32)) : 0.0;
          const double z = block_scan<2>(w, above, sh.scan);
          double* by_rank = reinterpret_cast<double*>(dyn) + kList;
          if (tid == 0) sh.at = 0;
          __syncthreads();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = 2 * tid + i;
            if (r >= m1) continue;
            by_rank[r] = w[i];
            // both cuts keep a first part of the ranks, the first rank always
            if (r == 0 || ((!cut_p || above[i] <= p * z) && w[i] >= min_p)) atomicMax(&sh.at, (uint32_t)r + 1u);
          }
          __syncthreads();
          const int kept = (int)sh.at, size = pow2_from(kept);
          uint64_t mine[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = 2 * tid + i;
            mine[i] = r < kept ? (list[r] << 32 | (uint32_t)r) : 0;  // the low half rises as the index falls
          }
          __syncthreads();
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (2 * tid + i < size) list[2 * tid + i] = mine[i];
          sort_down(list, size);
#pragma unroll
          for (int i = 0; i < 2; ++i) w[i] = 2 * tid + i < kept ? by_rank[(uint32_t)list[2 * tid + i]] : 0.0;
          const double mass = block_scan<2>(w, above, sh.scan);
          const double target = u * mass;
          if (tid == 0) sh.pick = kept - 1;  // when rounding lets none pass
          __syncthreads();
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (2 * tid + i < kept && above[i] + w[i] > target) atomicMin(&sh.pick, 2 * tid + i);
          __syncthreads();
          if (tid == 0) a.out[m] = (int64_t)(0xffffffffu - (uint32_t)(list[sh.pick] >> 32));
        }
        cluster_sync();  // no CTA leaves while another reads its shared memory
        return;
      }
    }
  } else if (cut_p && !cut_k && binned) {
    const double zc = row.template histogram<false>();
    if (tid == 0) sh.x_mass = zc, sh.at = kHist;
    cluster_sync();
    double z = 0.0;
    for (uint32_t r = 0; r < nc; ++r) z += remote_f64(&sh.x_mass, r);
    const double target = p * z;
    double v[2], before[2];
    row.row_bins(v);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v[i] *= 0x1p-15 * exp_tab(-(double)(2 * tid + i), kTable / 0.6931471805599453 / kPerNat, 1.0 / kPerNat, sh.tab);
    block_scan<2>(v, before, sh.scan);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (before[i] <= target && before[i] + v[i] > target) atomicMin(&sh.at, 2u * tid + i);
    __syncthreads();
    const uint32_t at = sh.at;
    if (at < kHist) {
      const float w0 = at > 0 ? (float)(at - 1) : 0.0f, w1 = (float)(at + 2);
      row.gather(w0, w1);
      double above = 0.0;
      row.each([&](uint32_t k, int) {
        if (k != 0 && row.depth(k) < w0) above += row.weight(k);
      });
      above = block_sum(above, sh.scan);
      if (tid == 0) sh.x_above = above;
      cluster_sync();
      if (rank == 0) {
        uint64_t* list = reinterpret_cast<uint64_t*>(dyn);
        const int total = row.collect();
        if (tid == 0) sh.x_keep = 0, sh.at = 0;
        if (total > 0) {
          double base = 0.0;
          for (uint32_t r = 0; r < nc; ++r) base += remote_f64(&sh.x_above, r);
          double w[4], before4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = 4 * tid + i < total ? row.weight((uint32_t)(list[4 * tid + i] >> 32)) : 0.0;
          const double inside = block_scan<4>(w, before4, sh.scan);
          __syncthreads();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (4 * tid + i < total && base + before4[i] <= target) atomicMax(&sh.at, 4u * tid + i + 1u);
          __syncthreads();
          const uint32_t kept = sh.at;  // of the list; the cut lies inside it when its ends say so
          if (kept > 0 && base + inside > target) {
            const uint32_t key = (uint32_t)(list[kept - 1] >> 32);
            uint32_t same = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              same += 4u * tid + i < kept && (uint32_t)(list[4 * tid + i] >> 32) == key ? 1u : 0u;
            same = __reduce_add_sync(0xffffffffu, same);
            if (lane == 0 && same) atomicAdd(&sh.x_keep, same);
            if (tid == 0) sh.x_key = key;
          }
        }
      }
      cluster_sync();
      const uint32_t keep = remote_u32(&sh.x_keep, 0);
      if (keep > 0) {
        ckey = remote_u32(&sh.x_key, 0);
        cties = keep;
        digits = false;
      }
    }
  }
  if (digits) {
    uint32_t alone = 0;
    double alone_w = 0.0;
    if (cut_k) {
      const auto c = row.template select<true>(klo, (double)(top_k - 1), 0u, 0.0);
      ckey = c.key;
      const double keep = (double)top_k - c.base;  // of c.mass ties
      cties = (uint32_t)(keep < c.mass ? keep : c.mass);
      alone = ckey;
      alone_w = (double)cties * row.weight(ckey);
    }
    if (cut_p) {
      const auto c = row.template select<false>(ckey, p, alone, alone_w);
      const double w = row.weight(c.key);
      const uint32_t all = (uint32_t)rint(c.mass / w);
      const double more = floor((c.target - c.base) / w);
      ckey = c.key;
      cties = more + 1.0 < (double)all ? (uint32_t)more + 1u : all;
    }
  }

  // kept weight above the cut and ties at it, per contiguous segment of a thread
  // (odd lengths, so that the threads of a warp start in different banks)
  const int seg = ((n + kThreads - 1) / kThreads) | 1;
  const int s0 = min(tid * seg, n), s1 = min(s0 + seg, n);
  double w_tie = row.weight(ckey);
  if (w_tie < min_p) w_tie = 0.0;
  double strict = 0.0;
  uint32_t ties = 0;
  for (int i = s0; i < s1; ++i) {
    const uint32_t k = keys[i];
    if (k > ckey) {
      const double w = row.weight(k);
      strict += w >= min_p ? w : 0.0;
    } else if (k == ckey) {
      ++ties;
    }
  }
  // ties before each thread (exclusive, in this CTA) and the CTA's sums
  uint32_t it = ties;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) it += v;
  }
  double st = strict;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) st += __shfl_xor_sync(0xffffffffu, st, o);
  if (lane == 31) sh.iscan[warp] = it;
  if (lane == 0) sh.scan[warp] = st;
  __syncthreads();
  uint32_t before = it - ties;
  for (int w = 0; w < warp; ++w) before += sh.iscan[w];
  if (tid == 0) {
    double s = 0.0;
    uint32_t t = 0;
    for (int w = 0; w < kWarps; ++w) s += sh.scan[w], t += sh.iscan[w];
    sh.x_mass = s;
    sh.x_ties = t;
  }
  cluster_sync();
  // every CTA finds the one that holds the target
  double off[kMaxCluster + 1];
  uint32_t my_before = 0, tb = 0;
  off[0] = 0.0;
  for (uint32_t r = 0; r < nc; ++r) {
    const uint32_t t = remote_u32(&sh.x_ties, r);
    if (r == rank) my_before = tb;
    const uint32_t kept = tb < cties ? min(t, cties - tb) : 0u;
    off[r + 1] = off[r] + (remote_f64(&sh.x_mass, r) + (double)kept * w_tie);
    tb += t;
  }
  const double target = u * off[nc];
  uint32_t owner = 0;
  for (uint32_t r = 0; r < nc; ++r)
    if (off[r + 1] > off[r] && off[r] <= target) owner = r;
  if (owner == rank) {
    const double local = target - off[rank];
    before += my_before;
    const uint32_t mine = before < cties ? min(ties, cties - before) : 0u;
    const double mass = strict + (double)mine * w_tie;
    double incl = mass;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) sh.scan[warp] = incl;
    __syncthreads();
    double wb = 0.0;
    for (int w = 0; w < warp; ++w) wb += sh.scan[w];
    double excl = __shfl_up_sync(0xffffffffu, incl, 1);
    excl = lane == 0 ? wb : wb + excl;
    // the first thread whose running sum passes the target; when rounding lets
    // none pass, the last one with any weight
    if (wb + incl > local && mass > 0.0) atomicMin(&sh.pick, tid);
    __syncthreads();
    if (sh.pick == kThreads) {
      __syncthreads();
      if (tid == 0) sh.pick = -1;
      __syncthreads();
      if (mass > 0.0) atomicMax(&sh.pick, tid);
      __syncthreads();
    }
    if (tid == sh.pick) {
      double c = excl;
      int at = s0;
      uint32_t tie = before;
      for (int i = s0; i < s1; ++i) {
        const uint32_t k = keys[i];
        double w = 0.0;
        if (k > ckey) {
          w = row.weight(k);
          w = w >= min_p ? w : 0.0;
        } else if (k == ckey) {
          w = tie < cties ? w_tie : 0.0;
          ++tie;
        }
        if (w > 0.0) {
          at = i;
          c += w;
          if (c > local) break;
        }
      }
      a.out[m] = lo + at;
    }
  }
  cluster_sync();  // no CTA leaves while another reads its shared memory
}

constexpr int kSmemMax = 200 * 1024;  // dynamic, beside the static struct

template <typename T>
int launch_filter(FilterArgs a, int64_t rows, cudaStream_t st) {
  constexpr int per = (kSmemMax - kWorkBytes) / (int)sizeof(typename KeyOf<T>::K) / 8 * 8;
  // CTAs of a row: as many as leave two places an SM (by shared memory), and up to 8
  // while the rows alone leave SMs idle
  constexpr int two = (110 * 1024 - kWorkBytes - (int)sizeof(Shared)) / (int)sizeof(typename KeyOf<T>::K);
  int nc = 1;
  while (nc < kMaxCluster && ((a.V + nc - 1) / nc > two || rows * nc <= 148)) nc *= 2;
  const int64_t chunk = ((a.V + nc - 1) / nc + 7) / 8 * 8;
  if (chunk > per) return CSAQ_ERR_UNSUPPORTED;
  a.chunk = (int)chunk;
  if (rows * nc > INT32_MAX) return CSAQ_ERR_UNSUPPORTED;
  auto kern = sample_filter_kernel<T>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel's shared memory is set
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64)) return CSAQ_ERR_UNSUPPORTED;
  if (e == cudaSuccess && !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * nc));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kWorkBytes + chunk * sizeof(typename KeyOf<T>::K);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = nc;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kern, a);
  }
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    (void)cudaGetLastError();
    return CSAQ_ERR_CUDA;
  }
  return launch_status();
}

}  // namespace
}  // namespace csaq

using namespace csaq;

extern "C" int csaq_sample_filtered(const void* logits, int n_parts, int64_t part_stride, int64_t ld, int64_t part_len,
                                    int64_t rows, const csaq_sample_params* params, const float* random, int64_t* out,
                                    int dtype, void* stream) {
  if (!logits || !params || !random || !out || n_parts < 1 || part_len < 1 || rows < 0 || ld < part_len ||
      (n_parts > 1 && part_stride < 0))
    return CSAQ_ERR_ARG;
  if (dtype != CSAQ_DT_F16 && dtype != CSAQ_DT_BF16 && dtype != CSAQ_DT_F32) return CSAQ_ERR_ARG;
  if (part_len > (1 << 30) || n_parts > (1 << 20) || (int64_t)n_parts * part_len > (1 << 30)) return CSAQ_ERR_UNSUPPORTED;
  if (rows == 0) return CSAQ_OK;
  const FilterArgs a{logits, n_parts, n_parts == 1 ? 0 : part_stride, ld, part_len, n_parts * part_len, *params,
                     random, out, 0};
  cudaStream_t st = as_stream(stream);
  if (dtype == CSAQ_DT_BF16) return launch_filter<__nv_bfloat16>(a, rows, st);
  if (dtype == CSAQ_DT_F16) return launch_filter<__half>(a, rows, st);
  return launch_filter<float>(a, rows, st);
}
