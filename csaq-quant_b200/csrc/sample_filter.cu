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
// some of them across u. Sums are therefore fp64, weights good to 2^-32 and a function
// of the key alone (their errors, one per value and of either sign, move a border by
// some 1e-11), and no sum goes through an atomic: every order is fixed.
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
#include <cfloat>

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

// Keys order like the logits, -0 and +0 as one value. kLow is -inf's: a key up to it is
// -inf or a negative NaN's, one above kInf a positive NaN's (those are set to 0 before
// use). keys(w): of the packed logits of a 32-bit word.
template <typename T> struct KeyOf;
template <> struct KeyOf<float> {
  using K = uint32_t;
  static constexpr uint32_t kLow = 0x007fffffu, kInf = 0xff800000u;
  static __device__ __forceinline__ uint32_t keys(uint32_t w) {
    const int b = __float_as_int(__uint_as_float(w) + 0.0f);
    return (uint32_t)b ^ ((uint32_t)(b >> 31) | 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  }
  static __device__ __forceinline__ uint32_t max_in(uint32_t k) { return k; }  // of the keys of a word
  static __device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) { return max(a, b); }
};
struct Key16 {
  using K = uint16_t;
  static __device__ __forceinline__ uint32_t ordered(uint32_t w) {
    return w ^ (((w >> 15) & 0x00010001u) * 0x7fffu | 0x80008000u);
  }
  static __device__ __forceinline__ uint32_t max_in(uint32_t k) { return max(k & 0xffffu, k >> 16); }
  static __device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
};
template <> struct KeyOf<__half> : Key16 {
  static constexpr uint32_t kLow = 0x03ffu, kInf = 0xfc00u;
  static __device__ __forceinline__ uint32_t keys(uint32_t w) {
    const __half2 r = __hadd2(*reinterpret_cast<__half2*>(&w), __float2half2_rn(0.0f));
    return ordered(*reinterpret_cast<const uint32_t*>(&r));
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __half2float(__ushort_as_half((unsigned short)(k & 0x8000u ? k & 0x7fffu : ~k)));
  }
};
template <> struct KeyOf<__nv_bfloat16> : Key16 {
  static constexpr uint32_t kLow = 0x007fu, kInf = 0xff80u;
  static __device__ __forceinline__ uint32_t keys(uint32_t w) {
    const __nv_bfloat162 r = __hadd2(*reinterpret_cast<__nv_bfloat162*>(&w), __float2bfloat162_rn(0.0f));
    return ordered(*reinterpret_cast<const uint32_t*>(&r));
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float((k & 0x8000u ? k & 0x7fffu : ~k & 0xffffu) << 16);
  }
};
template <typename T>
__device__ __forceinline__ typename KeyOf<T>::K key_of(T v) {
  return (typename KeyOf<T>::K)KeyOf<T>::keys(bits_of<T>(v));
}

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

// exp((v - x) / T) for a result of at least exp(kNegligible), with ch + cl = 256 / (T ln 2):
// table-driven reduction (Tang 1989) in pairs of fp32. (v - x) exactly as d + e, its
// product with ch + cl as n + f with n whole; exp = 2^(n / 256) (1 + r + r^2 / 2 + r^3 / 6),
// r = f ln 2 / 256, |r| <= 0.00136. r is good to 2^-34 and so is the bracket; fp64 takes only
// the last step (measured here at 12000 clocks for 16000 weights a CTA when it took all).
__device__ __forceinline__ double exp_tab(float v, float x, float ch, float cl, const double* tab) {
  const float d = v - x, dv = d - v, e = (v - (d - dv)) - (x + dv);
  const float zh = d * ch;
  const float zl = fmaf(e, ch, fmaf(d, cl, fmaf(d, ch, -zh)));
  const float magic = 12582912.0f;  // 1.5 2^23: the sum's low bits are the rounded integer
  const float t = zh + magic;
  const int n = __float_as_int(t) - __float_as_int(magic);
  const float r = ((zh - (t - magic)) + zl) * 0.0027076061740622863f;
  const float q = fmaf(r * r, fmaf(r, 1.0f / 6.0f, 0.5f), r);
  const double c = tab[n & (kTable - 1)];
  const double w = fma(c, widen(q), c);
  return __hiloint2double(__double2hiint(w) + ((n >> 8) << 20), __double2loint(w));
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
  uint32_t x_min, x_top;  // read by others: smallest and largest key of a window, or the first index
  uint32_t x_count;  // read by others: tokens in this CTA's list
  uint32_t x_key, x_keep;  // read by others (CTA 0): the cut of a nucleus; x_keep 0: none was found
  uint32_t wmax[kWarps];
  int pick;
  uint32_t at;
  __align__(8) uint32_t hist[kHist];  // read by others
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
  float fmax, ch, cl, lowest, per_bin;  // largest logit, 256 / (T ln 2), the lowest logit with weight, bins
  uint32_t kmax;

  // (no branch: the weights of a piece are computed side by side)
  __device__ __forceinline__ double weight(uint32_t k) const {
    const float v = KO::value(k);
    const double w = exp_tab(v, fmax, ch, cl, sh->tab);
    return v >= lowest ? w : 0.0;
  }
  // bins below the largest logit, in exact order of the keys; kHist and more: none
  __device__ __forceinline__ float depth(uint32_t k) const { return (fmax - KO::value(k)) * per_bin; }

  static constexpr int PER = 16 / (int)sizeof(K);  // keys of a 16-byte piece
  // f(keys, position, count) over 16-byte pieces (the last one may hold fewer keys);
  // pieces without a key from `from` on are passed over
  template <typename F>
  __device__ __forceinline__ void pieces(uint32_t from, F f) const {
    for (int i = threadIdx.x * PER; i < n; i += kThreads * PER) {
      const uint4 u = *reinterpret_cast<const uint4*>(keys + i);  // the buffer ends with a whole piece
      const int count = min(PER, n - i);
      if (KO::max_in(KO::max_of(KO::max_of(u.x, u.y), KO::max_of(u.z, u.w))) < from && count == PER) continue;
      const K* e = reinterpret_cast<const K*>(&u);
      uint32_t k[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) k[j] = j < count ? (uint32_t)e[j] : 0u;
      f(k, i);
    }
  }
  // f(key, position) over the keys from `from` (at least 1) on
  template <typename F>
  __device__ __forceinline__ void each(uint32_t from, F f) const {
    pieces(from, [&](const uint32_t (&k)[PER], int i) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (k[j] >= from) f(k[j], i + j);
    });
  }

  struct Cut {
    uint32_t key;   // lowest kept key
    double base;    // weight ranked above it
    double mass;    // weight at it
    double target;  // the bound that the weight ranked above a kept element meets
  };

  // The lowest-ranked element whose weight ranked above is at most the target, among
  // keys in [klo, khi], with weight `base` ranked above all of them; keys of `alone`
  // count once, with weight `alone_w` (nothing when 0). COUNT: weights 1. REL: the target
  // is `bound` times the keys' weight, else `bound`.
  template <bool COUNT, bool REL>
  __device__ Cut select(uint32_t klo, uint32_t khi, double base, double bound, uint32_t alone, double alone_w) {
    double* hist = reinterpret_cast<double*>(work);  // [bin][thread]
    const uint32_t span = khi - klo;
    const int bits = 32 - __clz(span | 1u);
    uint32_t prefix = 0;
    Cut c{klo, base, 0.0, bound};
    bool first_pass = true;
    __syncthreads();
    for (int shift = (bits - 1) / kDigit * kDigit; shift >= 0; shift -= kDigit) {
#pragma unroll
      for (int b = 0; b < kBins; ++b) hist[b * kThreads + threadIdx.x] = 0.0;
      each(klo, [&](uint32_t k, int) {
        const uint32_t o = k - klo;
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
      if (first_pass && REL) {
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

  // The row's histogram, bins 2 t and 2 t + 1 of thread t (after a cluster_sync).
  __device__ __forceinline__ void row_bins(double (&v)[2]) const {
    v[0] = v[1] = 0.0;
    for (uint32_t r = 0; r < nc; ++r) {
      const uint64_t x = remote_u64(reinterpret_cast<const uint64_t*>(sh->hist) + threadIdx.x, r);
      v[0] += (double)(uint32_t)x;
      v[1] += (double)(uint32_t)(x >> 32);
    }
  }
  // The element at `position` with key k into this CTA's list; sh->x_count of them, or
  // more than it holds.
  __device__ __forceinline__ void put(uint32_t k, int position) {
    const uint32_t at = atomicAdd(&sh->x_count, 1u);
    if (at < (uint32_t)kList)
      reinterpret_cast<uint64_t*>(work)[at] = (uint64_t)k << 32 | (0xffffffffu - (uint32_t)(first + position));
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
static_assert(kHist * 8 * 4 <= kBins * kThreads * 8, "the copies of the bins share the work area");
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

  for (int i = tid; i < kHist; i += kThreads) sh.hist[i] = 0;
  if (tid == 0) sh.x_count = 0, sh.at = kHist, sh.x_min = 0xffffffffu, sh.x_top = 0;

  // the slice as keys, and the thread's largest
  uint32_t tmax = 0;
  constexpr int VE = 16 / (int)sizeof(T);
  const T* base = reinterpret_cast<const T*>(a.logits) + m * a.ld;
  const bool vec = reinterpret_cast<uintptr_t>(base) % 16 == 0 && a.part_len % VE == 0 && a.part_stride % VE == 0;
  int done = 0;
  if (vec) {
    const int pieces = n / VE;
    for (int i0 = tid; i0 < pieces; i0 += 4 * kThreads) {
      uint4 u[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = i0 + q * kThreads;
        if (i < pieces) {
          const int64_t j = lo + (int64_t)i * VE, r = a.n_parts == 1 ? 0 : j / a.part_len;
          u[q] = __ldcs(reinterpret_cast<const uint4*>(base + r * a.part_stride + (j - r * a.part_len)));
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = i0 + q * kThreads;
        if (i < pieces) {
          u[q] = make_uint4(KO::keys(u[q].x), KO::keys(u[q].y), KO::keys(u[q].z), KO::keys(u[q].w));
          reinterpret_cast<uint4*>(keys)[i] = u[q];
          tmax = KO::max_of(tmax, KO::max_of(KO::max_of(u[q].x, u[q].y), KO::max_of(u[q].z, u[q].w)));
        }
      }
    }
    tmax = KO::max_in(tmax);
    done = pieces * VE;
  }
  for (int i = done + tid; i < n; i += kThreads) {
    const int64_t j = lo + i, r = a.n_parts == 1 ? 0 : j / a.part_len;
    const K k = key_of<T>(base[r * a.part_stride + (j - r * a.part_len)]);
    keys[i] = k;
    tmax = max(tmax, (uint32_t)k);
  }
  auto row_max = [&]() {  // the largest key of the row
    uint32_t v = __reduce_max_sync(0xffffffffu, tmax);
    if (lane == 0) sh.wmax[warp] = v;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; ++w) v = max(v, sh.wmax[w]);
      sh.x_max = v;
    }
    cluster_sync();
    v = 0;
    for (uint32_t r = 0; r < nc; ++r) v = max(v, remote_u32(&sh.x_max, r));
    return v;
  };
  uint32_t kmax = row_max();
  if (kmax > KO::kInf) {  // a NaN somewhere: out with them
    cluster_sync();
    tmax = 0;
    for (int i = tid; i < n; i += kThreads) {
      if (keys[i] > KO::kInf) keys[i] = 0;
      tmax = max(tmax, (uint32_t)keys[i]);
    }
    kmax = row_max();
  }
  if (kmax == KO::kInf) {  // +inf: its like share everything, as zeros among nothing
    cluster_sync();
    const K zero = key_of<T>(from_f32<T>(0.0f));
    tmax = 0;
    for (int i = tid; i < n; i += kThreads) {
      keys[i] = keys[i] == KO::kInf ? zero : (K)0;
      tmax = max(tmax, (uint32_t)keys[i]);
    }
    kmax = row_max();
  }
  if (kmax <= KO::kLow) {  // nothing to draw, for every CTA of the row
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
  if (!(min_p > 0.0)) min_p = 0.0;
  if (min_p > 1.0) min_p = 1.0;
  if (!(u > 0.0)) u = 0.0;
  if (u >= 1.0) u = 1.0 - 0x1p-53;

  Row<T> row;
  row.keys = keys, row.n = n, row.first = lo, row.sh = &sh, row.work = dyn, row.rank = rank, row.nc = nc, row.parity = 0;
  row.kmax = kmax;
  const float xmax = KO::value(kmax);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)fminf(fmaxf(temp, 1e-30f), 1e30f), c256 = inv_t * (kTable / 0.6931471805599453);
  row.fmax = xmax;
  row.ch = (float)c256;
  row.cl = (float)(c256 - (double)row.ch);
  const double x_low = (double)xmax + kNegligible / inv_t;
  row.lowest = x_low > -3.4e38 ? (float)x_low : -FLT_MAX;
  row.per_bin = fminf((float)(inv_t * kPerNat), 1e30f);

  // the lowest key that can have weight: a little below max + kNegligible T
  const double x_klo = x_low - 1.0 / inv_t;
  uint32_t klo = x_klo > -3.0e38 ? (uint32_t)key_of<T>(from_f32<T>((float)(x_klo - fabs(x_klo) * 0x1p-6))) : 0u;
  klo = klo <= KO::kLow ? KO::kLow + 1 : (klo > kmax ? kmax : klo);

  if (greedy) {  // the first index of the largest logit
    uint32_t at = 0xffffffffu;
    row.each(kmax, [&](uint32_t, int i) { at = min(at, (uint32_t)(lo + i)); });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) atomicMin(&sh.x_min, at);
    cluster_sync();
    if (rank == 0 && tid == 0) {
      for (uint32_t r = 0; r < nc; ++r) at = min(at, remote_u32(&sh.x_min, r));
      a.out[m] = at;
    }
    cluster_sync();
    return;
  }
  const bool cut_k = top_k > 0 && top_k < a.V, cut_p = top_p < 1.0f && !greedy;  // a NaN top_p switches it off
  const double p = top_p > 0.0f ? (double)top_p : 0.0;
  // keys above ckey are kept, and the first cties of those at it
  uint32_t ckey = klo, cties = 0xffffffffu;
  bool digits = cut_k || cut_p;
  // where a difference of logits that overflows is out of the bins' range in truth, too
  const bool binned = fabsf(xmax) <= 1e38f;

  if (cut_k && top_k <= kListK && binned) {
    // The k-th largest of the threads' largest keys has k elements from it on, and few
    // more when the large ones are spread over the row: a histogram of one key a thread.
    const float u0 = tmax >= klo ? row.depth(tmax) : (float)kHist;
    const int bin = u0 < (float)kHist ? (int)u0 : kHist;
    if (bin < kHist) atomicAdd(&sh.hist[bin], 1u);
    cluster_sync();
    double v[2], before[2];
    row.row_bins(v);
    block_scan<2>(v, before, sh.scan);
#pragma unroll
    for (int i = 0; i < 2; ++i)  // the bin that the k-th of them falls into
      if (before[i] < (double)top_k && before[i] + v[i] >= (double)top_k) sh.at = 2 * tid + i;
    __syncthreads();
    const uint32_t at = sh.at;
    if (at < kHist) {
      if (bin == (int)at) atomicMin(&sh.x_min, tmax);
      cluster_sync();
      uint32_t from = 0xffffffffu, total = 0;
      for (uint32_t r = 0; r < nc; ++r) from = min(from, remote_u32(&sh.x_min, r));
      row.each(from, [&](uint32_t k, int i) { row.put(k, i); });
      cluster_sync();
      for (uint32_t r = 0; r < nc; ++r) total += remote_u32(&sh.x_count, r);
      klo = from;  // at least k elements from here on
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
    // this CTA's masses per bin, as 2^15 w / 2^-bin (bin in nats / kPerNat), and the exact sum
    double zc = 0.0;
    // (eight copies of a bin, so that lanes with one logit seldom meet)
    uint32_t* copies = reinterpret_cast<uint32_t*>(dyn);
    for (int i = tid; i < kHist * 8 / 4; i += kThreads) reinterpret_cast<uint4*>(copies)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    row.pieces(klo, [&](const uint32_t (&k)[Row<T>::PER], int) {
#pragma unroll
      for (int j0 = 0; j0 < Row<T>::PER; j0 += 4) {
        double w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = row.weight(k[j0 + j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          zc += k[j0 + j] >= klo ? w[j] : 0.0;
          const float d = row.depth(k[j0 + j]);
          if (k[j0 + j] >= klo && d < (float)kHist) {
            const int b = (int)d;
            atomicAdd(&copies[b * 8 + (lane & 7)], (uint32_t)(32768.0f * __expf(((float)b - d) * (1.0f / kPerNat))));
          }
        }
      }
    });
    __syncthreads();
    for (int i = tid; i < kHist; i += kThreads) {
      const uint4 x = reinterpret_cast<const uint4*>(copies)[2 * i], y = reinterpret_cast<const uint4*>(copies)[2 * i + 1];
      sh.hist[i] = x.x + x.y + x.z + x.w + y.x + y.y + y.z + y.w;
    }
    zc = block_sum(zc, sh.scan);
    if (tid == 0) sh.x_mass = zc;
    cluster_sync();
    double z = 0.0;
    for (uint32_t r = 0; r < nc; ++r) z += remote_f64(&sh.x_mass, r);
    const double target = p * z;
    double v[2], before[2];
    row.row_bins(v);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v[i] *= 0x1p-15 * (double)__expf(-(float)(2 * tid + i) * (1.0f / kPerNat));
    block_scan<2>(v, before, sh.scan);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (before[i] <= target && before[i] + v[i] > target) atomicMin(&sh.at, 2u * tid + i);
    __syncthreads();
    const uint32_t at = sh.at;
    if (at < kHist) {
      const float w0 = at > 0 ? (float)(at - 1) : 0.0f, w1 = (float)(at + 2);
      double above = 0.0;
      uint32_t wlo = 0xffffffffu, whi = 0;
      row.each(klo, [&](uint32_t k, int i) {
        const float d = row.depth(k);
        if (d < w0) {
          above += row.weight(k);
        } else if (d < w1) {
          row.put(k, i);
          wlo = min(wlo, k);
          whi = max(whi, k);
        }
      });
      wlo = __reduce_min_sync(0xffffffffu, wlo);
      whi = __reduce_max_sync(0xffffffffu, whi);
      if (lane == 0) atomicMin(&sh.x_min, wlo), atomicMax(&sh.x_top, whi);
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
      } else {  // too many for the list: the digits of the window alone
        uint32_t total = 0;
        double sum = 0.0;
        wlo = 0xffffffffu, whi = 0;
        for (uint32_t r = 0; r < nc; ++r) {
          total += remote_u32(&sh.x_count, r);
          sum += remote_f64(&sh.x_above, r);
          wlo = min(wlo, remote_u32(&sh.x_min, r));
          whi = max(whi, remote_u32(&sh.x_top, r));
        }
        if (total > (uint32_t)kList && sum <= target) {
          const auto c = row.template select<false, false>(wlo, whi, sum, target, 0u, 0.0);
          if (c.key > wlo || c.base + c.mass > target) {  // the cut is not below the window
            const double w = row.weight(c.key), all = rint(c.mass / w), more = floor((target - c.base) / w) + 1.0;
            ckey = c.key;
            cties = (uint32_t)(more < all ? more : all);
            digits = false;
          }
        }
      }
    }
  }
  if (digits) {
    uint32_t alone = 0;
    double alone_w = 0.0;
    if (cut_k) {
      const auto c = row.template select<true, false>(klo, kmax, 0.0, (double)(top_k - 1), 0u, 0.0);
      ckey = c.key;
      const double keep = (double)top_k - c.base;  // of c.mass ties
      cties = (uint32_t)(keep < c.mass ? keep : c.mass);
      alone = ckey;
      alone_w = (double)cties * row.weight(ckey);
    }
    if (cut_p) {
      const auto c = row.template select<false, true>(cut_k ? ckey : klo, kmax, 0.0, p, alone, alone_w);
      const double w = row.weight(c.key);
      const uint32_t all = (uint32_t)rint(c.mass / w);
      const double more = floor((c.target - c.base) / w);
      ckey = c.key;
      cties = more + 1.0 < (double)all ? (uint32_t)more + 1u : all;
    }
  }

  // kept weight above the cut and ties at it, per contiguous segment of a thread: an odd
  // number of 16-byte pieces, so that neighbouring threads read from different banks
  constexpr int PER = Row<T>::PER;
  const int seg = (((n + PER - 1) / PER + kThreads - 1) / kThreads | 1) * PER;
  const int s0 = min(tid * seg, n), s1 = min(s0 + seg, n);
  double w_tie = row.weight(ckey);
  if (w_tie < min_p) w_tie = 0.0;
  double strict = 0.0;
  uint32_t ties = 0;
  for (int i = s0; i < s1; i += PER) {
    const uint4 piece = *reinterpret_cast<const uint4*>(keys + i);  // the buffer ends with a whole piece
    if (KO::max_in(KO::max_of(KO::max_of(piece.x, piece.y), KO::max_of(piece.z, piece.w))) < ckey && i + PER <= s1)
      continue;
    const K* e = reinterpret_cast<const K*>(&piece);
#pragma unroll
    for (int j0 = 0; j0 < PER; j0 += 4) {
      double w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = row.weight(e[j0 + j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = i + j0 + j < s1;
        strict += in && e[j0 + j] > ckey && w[j] >= min_p ? w[j] : 0.0;
        ties += in && e[j0 + j] == ckey ? 1u : 0u;
      }
    }
  }
  // ties before each thread (in this CTA) and the CTA's sums
  uint32_t it = ties;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) it += v;
  }
  const double strict_all = block_sum(strict, sh.scan);
  if (lane == 31) sh.iscan[warp] = it;
  __syncthreads();
  uint32_t before = it - ties, ties_all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t v = sh.iscan[w];
    before += w < warp ? v : 0u;
    ties_all += v;
  }
  if (tid == 0) {
    sh.x_mass = strict_all;
    sh.x_ties = ties_all;
    sh.pick = kThreads;
  }
  cluster_sync();
  // every CTA finds the one that holds the target: the last one that starts at or before
  // it (a lane per CTA)
  double start, all, target;
  uint32_t owner;
  {
    const bool is = lane < (int)nc;
    const uint32_t t = is ? remote_u32(&sh.x_ties, lane) : 0u;
    double mass = is ? remote_f64(&sh.x_mass, lane) : 0.0;
    uint32_t tb = t;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, tb, o);
      if (lane >= o) tb += v;
    }
    tb -= t;  // ties in the CTAs before
    mass += (double)(tb < cties ? min(t, cties - tb) : 0u) * w_tie;
    double incl = mass;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    double at = __shfl_up_sync(0xffffffffu, incl, 1);
    if (lane == 0) at = 0.0;
    all = __shfl_sync(0xffffffffu, incl, nc - 1);
    start = __shfl_sync(0xffffffffu, at, rank);
    before += __shfl_sync(0xffffffffu, tb, rank);
    target = u * all;
    owner = 31 - __clz(__ballot_sync(0xffffffffu, is && mass > 0.0 && at <= target));
  }
  if (owner == rank) {
    const double local = target - start;
    const uint32_t mine = before < cties ? min(ties, cties - before) : 0u;
    double mass[1] = {strict + (double)mine * w_tie}, excl[1];
    block_scan<1>(mass, excl, sh.scan);
    // the first thread whose running sum passes the target; when rounding lets
    // none pass, the last one with any weight
    if (excl[0] + mass[0] > local && mass[0] > 0.0) atomicMin(&sh.pick, tid);
    __syncthreads();
    if (sh.pick == kThreads) {
      __syncthreads();
      if (tid == 0) sh.pick = -1;
      __syncthreads();
      if (mass[0] > 0.0) atomicMax(&sh.pick, tid);
      __syncthreads();
    }
    if (warp == sh.pick / 32) {  // its warp goes through its segment, 32 elements at a time
      const int from = sh.pick % 32;
      const int a0 = __shfl_sync(0xffffffffu, s0, from), a1 = __shfl_sync(0xffffffffu, s1, from);
      double run = __shfl_sync(0xffffffffu, excl[0], from);
      uint32_t tie = __shfl_sync(0xffffffffu, before, from);
      int at = a0;
      for (int i0 = a0; i0 < a1; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t k = i < a1 ? (uint32_t)keys[i] : 0u;
        const uint32_t same = __ballot_sync(0xffffffffu, k == ckey);
        double w = row.weight(k);
        w = k > ckey && w >= min_p ? w : 0.0;
        if (k == ckey) w = tie + __popc(same & ((1u << lane) - 1u)) < cties ? w_tie : 0.0;
        tie += __popc(same);
        double incl = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        const uint32_t any = __ballot_sync(0xffffffffu, w > 0.0);
        const uint32_t past = __ballot_sync(0xffffffffu, w > 0.0 && run + incl > local);
        if (any) at = i0 + 31 - __clz(any);
        if (past) {
          at = i0 + __ffs(past) - 1;
          break;
        }
        run += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) a.out[m] = lo + at;
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
