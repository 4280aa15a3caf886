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
// some 1e-11), and no sum depends on an order: it is fixed, or the terms are integers.
//
// A cluster of CTAs takes one row and keeps it in shared memory: one pass over the
// logits. What follows depends on the row's settings:
//
//  list    top-k up to kListK: a histogram of counts over bins of 1/32 nat below the
//          largest logit says which bins hold the first k ranks; their tokens, little
//          more than k, are gathered in one CTA, sorted, cut and drawn from there.
//  nucleus top-p alone: a histogram of approximate masses says near which bin the cut
//          lies; one pass sums the exact weight of the row and of what lies above three
//          bins, whose tokens (no more than a list holds) are narrowed down to the cut,
//          1 / kHist of their keys' range at a time; the last pass adds those above it.
//  digits  anything else that cuts, and what the two above hand over (more tokens than
//          the list holds, a cut out of the bins' range): the cut is found three key
//          bits at a time; every thread adds its elements into 8 bins of its own, the
//          bins are summed in a fixed order over threads and CTAs, and the next pass
//          looks only at the bin that holds the cut.
//  none    no top-k, no top-p: the last pass alone.
//
// The histograms of 1/32 nat only say where to look; the answer never depends on them.
//
// Bound by the chain of phases between cluster barriers for few rows (1 x 128256 bf16:
// top-k 40 12.8 us, top-p 0.9 23), by those phases and instruction issue for many (64 x
// 151936: no filter 26 us, top-k 40 19, top-p 0.9 63, min-p 12, greedy 7.5; a copy of
// the logits would take 3): about 85 instructions a logit for a nucleus, 50 of them the
// weight, a third of its time.

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
constexpr int kTable = 256;            // 2^(j / 256)
constexpr double kNegligible = -50.0;  // weights under e^-50, 2e-22 of the largest, count as 0
constexpr uint32_t kAll = 0xffffffffu;
static_assert(kBins * 2 == kWarps && kList == 4 * kThreads && kHist == 2 * kThreads, "shares of a thread");
// The work area: a list, what its sort and its weights use, the histogram. Or the bins of
// the digit passes; or, for a nucleus, copies of the histogram and then the window's keys
// and their bins.
constexpr int kWorkBytes = kList * 8 + kThreads * 8 + kListK * 8, kAreaBytes = kWorkBytes + kHist * 4;
static_assert(kAreaBytes >= kBins * kThreads * 8 && kAreaBytes >= kHist * 8 * 4 && kWorkBytes >= kList * 4 + kHist * 16,
              "they share the area");

struct FilterArgs {
  const void* logits;
  int n_parts;
  int64_t part_stride, ld, part_len, V;
  csaq_sample_params p;
  const float* random;
  int64_t* out;
  int chunk;  // elements of a CTA's slice
};

// Logits of type T as they lie in 32-bit words. Comparisons go by value: -0 and +0 are
// one, a NaN is under everything. key(v) orders like v in as few bits as T has values;
// T's finite values start at kLowest or above.
template <typename T> struct Logit;
template <> struct Logit<float> {
  static constexpr int N = 1;
  static constexpr float kLowest = -FLT_MAX;
  static __device__ __forceinline__ float value(uint32_t w, int) { return __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float largest(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t key(float v) {
    const int b = __float_as_int(v + 0.0f);
    return (uint32_t)b ^ ((uint32_t)(b >> 31) | 0x80000000u);
  }
  static __device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  }
};
template <> struct Logit<__nv_bfloat16> {
  static constexpr int N = 2;
  static constexpr float kLowest = -FLT_MAX;
  static __device__ __forceinline__ float value(uint32_t w, int j) {
    return __uint_as_float(j ? w & 0xffff0000u : w << 16);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float largest(uint32_t w) { return fmaxf(value(w, 0), value(w, 1)); }
  static __device__ __forceinline__ uint32_t key(float v) { return Logit<float>::key(v) >> 16; }
  static __device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float((k & 0x8000u ? k & 0x7fffu : ~k & 0xffffu) << 16);
  }
};
template <> struct Logit<__half> {
  static constexpr int N = 2;
  static constexpr float kLowest = -65504.0f;
  static __device__ __forceinline__ float value(uint32_t w, int j) {
    return __half2float(__ushort_as_half((unsigned short)(j ? w >> 16 : w)));
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float largest(uint32_t w) { return fmaxf(value(w, 0), value(w, 1)); }
  static __device__ __forceinline__ uint32_t key(float v) {
    const uint32_t b = __half_as_ushort(__float2half_rn(v + 0.0f));
    return b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
  }
  static __device__ __forceinline__ float of_key(uint32_t k) {
    return __half2float(__ushort_as_half((unsigned short)(k & 0x8000u ? k & 0x7fffu : ~k)));
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
__device__ __forceinline__ uint64_t remote_u64(const void* p, uint32_t rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t remote_u32(const void* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
// one value of every CTA of the cluster, a lane each; `none` in the other lanes
__device__ __forceinline__ uint32_t each_u32(const uint32_t* p, uint32_t nc, uint32_t none) {
  const uint32_t lane = threadIdx.x & 31;
  return lane < nc ? remote_u32(p, lane) : none;
}
__device__ __forceinline__ double each_f64(const double* p, uint32_t nc) {
  const uint32_t lane = threadIdx.x & 31;
  return lane < nc ? __longlong_as_double((long long)remote_u64(p, lane)) : 0.0;
}
// the sum over the cluster in rank order
__device__ __forceinline__ double sum_f64(const double* p, uint32_t nc) {
  const double mine = each_f64(p, nc);
  double s = 0.0;
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r) s += __shfl_sync(0xffffffffu, mine, r);
  return s;
}

// exp((v - x) / T) for a result of at least exp(kNegligible), with ch + cl = 256 / (T ln 2):
// table-driven reduction (Tang 1989) in pairs of fp32. (v - x) as d + e, exact; its product
// with ch + cl as n + f with n whole; exp = 2^(n / 256) (1 + r + r^2 / 2 + r^3 / 6),
// r = f ln 2 / 256, |r| <= 0.00136. r is good to 2^-34 and so is the bracket; fp64 takes
// the last step alone. (e is not 0 for 16-bit logits either: those near 0 have bits below
// an fp32 difference from the largest, and half its step over T is the weight's error.)
__device__ __forceinline__ double exp_tab(float v, float x, float ch, float cl, const double* tab) {
  const float d = v - x, dv = d - v, e = (v - (d - dv)) - (x + dv);
  const float zh = d * ch;
  const float zl = fmaf(e, ch, fmaf(d, cl, fmaf(d, ch, -zh)));
  const float magic = 12582912.0f;  // 1.5 2^23: the sum's low bits are the rounded integer
  const float t = zh + magic;
  const int n = __float_as_int(t);  // and those of the magic number, which neither use below sees
  const float r = ((zh - (t - magic)) + zl) * 0.0027076061740622863f;
  const float q = fmaf(r * r, fmaf(r, 1.0f / 6.0f, 0.5f), r);
  const double c = tab[n & (kTable - 1)];
  const double w = fma(c, (double)q, c);
  // 2^(n / 256)'s whole part: n's bits from 8 on, into the exponent (from 20 on)
  return __hiloint2double(__double2hiint(w) + (int)(((uint32_t)n - 0x4b400000u & ~(kTable - 1u)) << 12),
                          __double2loint(w));
}

// Static shared memory; what other CTAs read is marked.
struct Shared {
  double tab[kTable];
  double red[2][kBins];  // read by others: this CTA's bin sums, alternating from pass to pass
  double tot[kBins];     // the row's
  double half[kWarps];
  double scan[kWarps];
  uint32_t iscan[kWarps];
  double x_mass;            // read by others
  double x_above;           // read by others
  uint32_t x_ties;          // read by others
  uint32_t x_max;           // read by others: the slice's largest logit, as a key
  uint32_t x_min, x_top;    // read by others: smallest and largest key of a window, or the first index
  uint32_t x_count;         // read by others: tokens in this CTA's list
  float wmax[kWarps];
  int pick;
  uint32_t at;
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
    const double x = warp_sums[w];
    if (w < warp) wb += x;
    all += x;
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

// Bitonic sort of n (a power of two, at most kList) in shared memory, largest first;
// `spare` holds kThreads. Up to a thread each they stay in registers, and neighbours up to
// 16 apart meet by shuffles.
__device__ __forceinline__ void sort_down(uint64_t* v, uint64_t* spare, int n) {
  __syncthreads();
  if (n <= kThreads) {
    const int i = threadIdx.x;
    uint64_t x = i < n ? v[i] : 0, *to = spare, *other = v;
    for (int size = 2; size <= n; size <<= 1)
      for (int step = size >> 1; step > 0; step >>= 1) {
        uint64_t y;
        if (step >= 32) {
          if (i < n) to[i] = x;
          __syncthreads();
          y = i < n ? to[i ^ step] : 0;
          uint64_t* const swap = to;
          to = other;
          other = swap;
        } else {
          y = __shfl_xor_sync(0xffffffffu, x, step);
        }
        const bool want_max = ((i & step) == 0) == ((i & size) == 0);
        x = (x < y) == want_max ? y : x;
      }
    __syncthreads();
    if (i < n) v[i] = x;
  } else {
    for (int size = 2; size <= n; size <<= 1)
      for (int step = size >> 1; step > 0; step >>= 1) {
        for (int i = threadIdx.x; i < n / 2; i += kThreads) {
          const int a = 2 * i - (i & (step - 1)), b = a + step;
          const uint64_t x = v[a], y = v[b];
          if ((x < y) == ((a & size) == 0)) v[a] = y, v[b] = x;
        }
        __syncthreads();
      }
  }
  __syncthreads();
}
__device__ __forceinline__ int pow2_from(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

template <typename T>
struct Row {
  using L = Logit<T>;
  static constexpr int PER = 16 / (int)sizeof(T);  // logits of a 16-byte piece
  const T* logits;  // the slice, in index order
  int n;
  int64_t first;  // index of its first element
  Shared* sh;
  uint8_t* work;  // kAreaBytes
  uint32_t rank, nc;
  int parity;
  float fmax, ch, cl, per_bin;  // largest logit, 256 / (T ln 2), bins per unit

  // (no branch: the weights of a piece are computed side by side; what lies under the
  // lowest logit with weight is for the caller to leave out)
  __device__ __forceinline__ double weight(float v) const {
    return exp_tab(v, fmax, ch, cl, sh->tab);
  }
  // bins below the largest logit, in the order of the logits; kHist and more: none
  __device__ __forceinline__ float depth(float v) const { return (fmax - v) * per_bin; }

  __device__ __forceinline__ static float top_of(const uint4& u) {
    return L::largest(L::larger(L::larger(u.x, u.y), L::larger(u.z, u.w)));
  }
  __device__ __forceinline__ static void values(const uint4& u, float (&v)[PER]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = L::value(w[j / L::N], j % L::N);
  }
  // f(values, position) over the 16-byte pieces of [i0, i1) with a logit from `from` on, a
  // piece every `step` elements; behind the slice's end values are NaN
  template <typename F>
  __device__ __forceinline__ void pieces(int i0, int i1, int step, float from, F f) const {
    for (int i = i0; i < i1; i += step) {
      const uint4 u = *reinterpret_cast<const uint4*>(logits + i);  // the buffer ends with a whole piece
      if (i + PER <= n && !(top_of(u) >= from)) continue;
      float v[PER];
      values(u, v);
      if (i + PER > n) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (i + j >= n) v[j] = __uint_as_float(0x7fffffffu);
      }
      f(v, i);
    }
  }
  // the same over the whole slice, pieces dealt to the threads in turn
  template <typename F>
  __device__ __forceinline__ void pieces(float from, F f) const {
    pieces(threadIdx.x * PER, n, kThreads * PER, from, f);
  }
  // f(logit, position) over the logits from `from` on
  template <typename F>
  __device__ __forceinline__ void each(float from, F f) const {
    pieces(from, [&](const float (&v)[PER], int i) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (v[j] >= from) f(v[j], i + j);
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
    const float from = L::of_key(klo);
    uint32_t prefix = 0;
    Cut c{klo, base, 0.0, bound};
    bool first_pass = true;
    __syncthreads();
    for (int shift = (bits - 1) / kDigit * kDigit; shift >= 0; shift -= kDigit) {
#pragma unroll
      for (int b = 0; b < kBins; ++b) hist[b * kThreads + threadIdx.x] = 0.0;
      each(from, [&](float v, int) {
        const uint32_t k = L::key(v), o = k - klo;
        if (o > span || (alone_w != 0.0 && k == alone) || (!first_pass && (o >> (shift + kDigit)) != prefix)) return;
        hist[((o >> shift) & (kBins - 1)) * kThreads + threadIdx.x] += COUNT ? 1.0 : weight(v);
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
      if (threadIdx.x < kBins * 32) {  // a warp a bin
        const double s = sum_f64(&sh->red[parity][threadIdx.x >> 5], nc);
        if ((threadIdx.x & 31) == 0) sh->tot[threadIdx.x >> 5] = s;
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

  // The row's sums of kHist bins, 2 t and 2 t + 1 for thread t (after a cluster_sync).
  __device__ __forceinline__ void row_bins(const uint64_t* bins, double (&v)[2]) const {
    uint64_t x[kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) x[r] = r < (int)nc ? remote_u64(bins + threadIdx.x, r) : 0;
    v[0] = v[1] = 0.0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      v[0] += (double)(uint32_t)x[r];
      v[1] += (double)(uint32_t)(x[r] >> 32);
    }
  }
  // select() among the keys that the CTAs have found (n in this one, at most kList), all in
  // [klo, khi] and in the order of 1 / kHist of that range at a time. A weight is added
  // as two integers of 20 bits, relative to the largest (2^-40, under its own error): the
  // sums do not depend on the order of the atomics.
  __device__ Cut narrow(const uint32_t* found, int n, uint32_t klo, uint32_t khi, double base, double bound) const {
    const double unit = weight(L::of_key(khi)) * 0x1p-40, per_unit = 1.0 / unit;
    uint64_t* bins = reinterpret_cast<uint64_t*>(work + kList * 4);  // low sums of two bins, high sums of two bins
    Cut c{klo, base, 0.0, bound};
    for (int flip = 0;; flip ^= 1) {
      const int shift = max(0, 22 - __clz(khi - klo | 1u));
      uint32_t* low = reinterpret_cast<uint32_t*>(bins + flip * kHist);
      for (int i = threadIdx.x; i < kHist; i += kThreads) low[i] = low[kHist + i] = 0;
      if (threadIdx.x == 0) sh->at = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t o = khi - found[i];
        if (o > khi - klo) continue;
        const uint64_t w = __double2ull_rn(fmin(weight(L::of_key(found[i])) * per_unit, 0x1p40));
        atomicAdd(&low[o >> shift], (uint32_t)w & 0xfffffu);
        atomicAdd(&low[kHist + (o >> shift)], (uint32_t)(w >> 20));
      }
      cluster_sync();
      double v[2], high[2], before[2];
      v[0] = v[1] = high[0] = high[1] = 0.0;
      if (2 * threadIdx.x <= khi - klo >> shift) {
        row_bins(reinterpret_cast<const uint64_t*>(low), v);
        row_bins(reinterpret_cast<const uint64_t*>(low + kHist), high);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) v[i] = (v[i] + high[i] * 0x1p20) * unit;
      block_scan<2>(v, before, sh->scan);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (v[i] > 0.0 && c.base + before[i] <= bound) atomicMax(&sh->at, 2 * threadIdx.x + i + 1);
      __syncthreads();
      const uint32_t pick = sh->at - 1;  // the first bin that holds a key is one
      if (threadIdx.x == pick / 2) sh->tot[0] = before[pick & 1], sh->tot[1] = v[pick & 1];
      __syncthreads();
      c.base += sh->tot[0];
      c.mass = sh->tot[1];
      khi -= pick << shift;
      if (shift == 0) {
        c.key = khi;
        return c;
      }
      klo = khi - klo >= 1u << shift ? khi - (1u << shift) + 1u : klo;
    }
  }
  // The element at `position` into this CTA's list; sh->x_count of them, or more than it
  // holds. Sorted downwards, an entry's order is that of the ranks.
  __device__ __forceinline__ void put(float v, int position) {
    const uint32_t at = atomicAdd(&sh->x_count, 1u);
    if (at < (uint32_t)kList)
      reinterpret_cast<uint64_t*>(work)[at] = (uint64_t)Logit<float>::key(v) << 32 | (kAll - (uint32_t)(first + position));
  }
  __device__ __forceinline__ static float logit_of(uint64_t entry) { return Logit<float>::of_key((uint32_t)(entry >> 32)); }
  // All lists in CTA 0, a warp a CTA; `total` (of all, at most kList). The other CTAs
  // are done with theirs at the next cluster_sync.
  __device__ void collect(uint32_t total) {
    uint64_t* list = reinterpret_cast<uint64_t*>(work);
    const uint32_t lane = threadIdx.x & 31, r = threadIdx.x >> 5;
    const uint32_t c = each_u32(&sh->x_count, nc, 0u);
    uint32_t before = c;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, before, o);
      if ((int)lane >= o) before += v;
    }
    before -= c;
    const uint32_t mine = __shfl_sync(0xffffffffu, c, r & 7), start = __shfl_sync(0xffffffffu, before, r & 7);
    if (r > 0 && r < nc)
      for (uint32_t i = lane; i < mine; i += 32) list[start + i] = remote_u64(list + i, r);
    for (int i = (int)total + threadIdx.x; i < pow2_from((int)total); i += kThreads) list[i] = 0;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_filter_kernel(const FilterArgs a) {
  using L = Logit<T>;
  constexpr int PER = Row<T>::PER;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Shared sh;
  const uint32_t rank = cluster_rank(), nc = cluster_size();
  const int64_t m = blockIdx.x / nc;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  T* slice = reinterpret_cast<T*>(dyn + kAreaBytes);
  const int64_t lo = (int64_t)rank * a.chunk;
  const int n = (int)(lo >= a.V ? 0 : (a.V - lo < a.chunk ? a.V - lo : a.chunk));
  if (tid < kTable) sh.tab[tid] = exp2((double)tid / kTable);
  uint32_t* const hist = reinterpret_cast<uint32_t*>(dyn + kWorkBytes);
  for (int i = tid; i < kHist; i += kThreads) hist[i] = 0;
  if (tid == 0) sh.x_count = 0, sh.at = kHist, sh.x_min = kAll, sh.x_top = 0;
  pdl_wait();
  pdl_trigger();

  // the slice, and the thread's largest logit
  float tmax = -INFINITY;
  const T* base = reinterpret_cast<const T*>(a.logits) + m * a.ld;
  const bool vec = reinterpret_cast<uintptr_t>(base) % 16 == 0 && a.part_len % PER == 0 && a.part_stride % PER == 0;
  int done = 0;
  if (vec) {
    const int whole = n / PER;
    for (int i0 = tid; i0 < whole; i0 += 4 * kThreads) {
      uint4 u[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = i0 + q * kThreads;
        if (i < whole) {
          const int64_t j = lo + (int64_t)i * PER, r = a.n_parts == 1 ? 0 : j / a.part_len;
          u[q] = __ldcs(reinterpret_cast<const uint4*>(base + r * a.part_stride + (j - r * a.part_len)));
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = i0 + q * kThreads;
        if (i < whole) {
          reinterpret_cast<uint4*>(slice)[i] = u[q];
          tmax = fmaxf(tmax, Row<T>::top_of(u[q]));
        }
      }
    }
    done = whole * PER;
  }
  for (int i = done + tid; i < n; i += kThreads) {
    const int64_t j = lo + i, r = a.n_parts == 1 ? 0 : j / a.part_len;
    const T x = base[r * a.part_stride + (j - r * a.part_len)];
    slice[i] = x;
    tmax = fmaxf(tmax, to_f32<T>(x));
  }
  auto row_max = [&]() {
    float v = tmax;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0) sh.wmax[warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = sh.wmax[lane % kWarps];
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
      if (lane == 0) sh.x_max = Logit<float>::key(v);
    }
    cluster_sync();
    return Logit<float>::of_key(__reduce_max_sync(0xffffffffu, each_u32(&sh.x_max, nc, 0u)));
  };
  float xmax = row_max();
  if (xmax == INFINITY) {  // +inf logits share everything: zeros among nothing
    cluster_sync();
    tmax = -INFINITY;
    for (int i = tid; i < n; i += kThreads) {
      const bool is = to_f32<T>(slice[i]) == INFINITY;
      slice[i] = from_f32<T>(is ? 0.0f : -INFINITY);
      if (is) tmax = 0.0f;
    }
    xmax = row_max();
  }
  if (xmax == -INFINITY) {  // nothing to draw, for every CTA of the row
    if (rank == 0 && tid == 0) a.out[m] = -1;
    cluster_sync();  // no CTA leaves while another reads its shared memory
    return;
  }
  const float temp = a.p.temperature ? a.p.temperature[m] : a.p.temperature_all;
  const int top_k = a.p.top_k ? a.p.top_k[m] : a.p.top_k_all;
  const float top_p = a.p.top_p ? a.p.top_p[m] : a.p.top_p_all;
  const float min_p = a.p.min_p ? a.p.min_p[m] : a.p.min_p_all;
  double u = a.random[m];
  if (!(u > 0.0)) u = 0.0;
  if (u >= 1.0) u = 1.0 - 0x1p-53;

  Row<T> row;
  row.logits = slice, row.n = n, row.first = lo, row.sh = &sh, row.work = dyn, row.rank = rank, row.nc = nc, row.parity = 0;
  row.fmax = xmax;
  if (!(temp > 0.0f)) {  // the first index of the largest logit
    uint32_t at = kAll;
    row.each(xmax, [&](float, int i) { at = min(at, (uint32_t)(lo + i)); });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) atomicMin(&sh.x_min, at);
    cluster_sync();
    at = __reduce_min_sync(0xffffffffu, each_u32(&sh.x_min, nc, kAll));
    if (rank == 0 && tid == 0) a.out[m] = at;
    cluster_sync();
    return;
  }
  const double t64 = fminf(fmaxf(temp, 1e-30f), 1e30f), c256 = kTable / 0.6931471805599453 / t64;
  row.ch = (float)c256;
  row.cl = (float)(c256 - (double)row.ch);
  row.per_bin = fminf((float)((double)kPerNat / t64), 1e30f);
  // The cut: logits above `cut` are kept, and the first `ties` of those at it. At first
  // it is the lowest logit with weight, or with min_p times the largest weight.
  const double limit = (double)xmax + t64 * (min_p > 0.0f ? log(fmin((double)min_p, 1.0)) : kNegligible);
  float lowest = (float)fmax(limit, -(double)FLT_MAX);
  if (min_p > 0.0f && (double)lowest < limit) lowest = nextafterf(lowest, INFINITY);
  const float negligible = (float)fmax((double)xmax + t64 * kNegligible, -(double)FLT_MAX);
  float cut = negligible;
  uint32_t ties = kAll;

  const bool cut_k = top_k > 0 && top_k < a.V, cut_p = top_p < 1.0f;  // a NaN top_p switches it off
  const double p = top_p > 0.0f ? (double)top_p : 0.0;
  bool digits = cut_k || cut_p;
  // A thread's contiguous segment for sums in index order: an odd number of 16-byte
  // pieces, so that neighbouring threads read from different banks.
  const int seg = (((n + PER - 1) / PER + kThreads - 1) / kThreads | 1) * PER;
  const int s0 = min(tid * seg, n), s1 = min(s0 + seg, n);
  double strict = 0.0;  // its weight above the window, when summed
  float window = 0.0f;  // the window's upper end, in bins
  bool summed = false;
  // where a difference of logits that overflows is out of the bins' range in truth, too
  const bool binned = fabsf(xmax) <= 1e38f;

  if (cut_k && top_k <= kListK && binned) {
    // The k-th largest of the threads' largest logits has k elements from it on, and few
    // more when the large ones are spread over the row: a histogram of one logit a thread.
    const float u0 = tmax >= negligible ? row.depth(tmax) : (float)kHist;
    const int bin = u0 < (float)kHist ? (int)u0 : kHist;
    if (bin < kHist) atomicAdd(&hist[bin], 1u);
    cluster_sync();
    double v[2], before[2];
    row.row_bins(reinterpret_cast<const uint64_t*>(hist), v);
    block_scan<2>(v, before, sh.scan);
#pragma unroll
    for (int i = 0; i < 2; ++i)  // the bin that the k-th of them falls into
      if (before[i] < (double)top_k && before[i] + v[i] >= (double)top_k) sh.at = 2 * tid + i;
    __syncthreads();
    const uint32_t at = sh.at;
    if (at < kHist) {
      if (bin == (int)at) atomicMin(&sh.x_min, Logit<float>::key(tmax));
      cluster_sync();
      const float from = Logit<float>::of_key(__reduce_min_sync(0xffffffffu, each_u32(&sh.x_min, nc, kAll)));
      row.each(from, [&](float x, int i) { row.put(x, i); });
      cluster_sync();
      const uint32_t total = __reduce_add_sync(0xffffffffu, each_u32(&sh.x_count, nc, 0u));
      cut = from;  // at least k elements from here on
      if (total <= (uint32_t)kList) {
        if (rank == 0) row.collect(total);
        cluster_sync();  // no CTA leaves while another reads its shared memory
        if (rank == 0) {
          uint64_t* list = reinterpret_cast<uint64_t*>(dyn);
          sort_down(list, list + kList, pow2_from((int)total));
          const int m1 = min((int)total, top_k);  // ranks 0 .. m1 - 1 pass top-k
          double w[2], above[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) w[i] = 2 * tid + i < m1 ? row.weight(Row<T>::logit_of(list[2 * tid + i])) : 0.0;
          const double z = block_scan<2>(w, above, sh.scan);
          double* by_rank = reinterpret_cast<double*>(dyn) + kList + kThreads;  // behind what a sort uses
          if (tid == 0) sh.at = 0;
          __syncthreads();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = 2 * tid + i;
            if (r >= m1) continue;
            by_rank[r] = w[i];
            // both cuts keep a first part of the ranks, the first rank always
            if (r == 0 || ((!cut_p || above[i] <= p * z) && Row<T>::logit_of(list[r]) >= lowest)) atomicMax(&sh.at, (uint32_t)r + 1u);
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
          sort_down(list, list + kList, size);
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
          if (tid == 0) a.out[m] = (int64_t)(kAll - (uint32_t)(list[sh.pick] >> 32));
        }
        return;
      }
    }
  } else if (cut_p && !cut_k && binned) {
    // masses per bin (the nearest whole depth), as 2^15 w / e^(-bin / kPerNat), in eight copies, so that
    // lanes with one logit seldom meet
    uint32_t* copies = reinterpret_cast<uint32_t*>(dyn);
    for (int i = tid; i < kHist * 8 / 4; i += kThreads) reinterpret_cast<uint4*>(copies)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    row.pieces(negligible, [&](const float (&x)[PER], int) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        // sums with 1.5 * 2^23 round, and leave the integer in the low bits
        const float d = row.depth(x[j]), t = d + 12582912.0f, r = ((t - 12582912.0f) - d) * (1.0f / kPerNat);
        const float mass = fmaf(fmaf(r, 0.5f, 1.0f) * r, 32768.0f, 32768.0f) + 12582912.0f;
        if (d < kHist - 1.0f)
          atomicAdd(&copies[(__float_as_int(t) - 0x4b400000) * 8 + (lane & 7)], __float_as_uint(mass) - 0x4b400000u);
      }
    });
    __syncthreads();
    uint32_t sums[2];  // (the last copies lie where the histogram goes)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = tid + j * kThreads;
      const uint4 x = reinterpret_cast<const uint4*>(copies)[2 * i], y = reinterpret_cast<const uint4*>(copies)[2 * i + 1];
      sums[j] = x.x + x.y + x.z + x.w + y.x + y.y + y.z + y.w;
    }
    __syncthreads();
    hist[tid] = sums[0], hist[tid + kThreads] = sums[1];
    cluster_sync();
    double v[2], before[2];
    row.row_bins(reinterpret_cast<const uint64_t*>(hist), v);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v[i] *= 0x1p-15 * (double)__expf(-(float)(2 * tid + i) * (1.0f / kPerNat));
    const double near = p * block_scan<2>(v, before, sh.scan);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (before[i] <= near && before[i] + v[i] > near) atomicMin(&sh.at, 2u * tid + i);
    __syncthreads();
    const uint32_t at = sh.at;
    if (at < kHist) {
      // exact weights, of everything and above the window
      window = at > 0 ? (float)at - 1.5f : 0.0f;
      const float w1 = (float)at + 1.5f;
      double zc = 0.0;
      uint32_t wlo = kAll, whi = 0, *found = reinterpret_cast<uint32_t*>(dyn);  // keys in the window
      row.pieces(s0, s1, PER, negligible, [&](const float (&x)[PER], int) {
uint32_t in = 0;  // which of the piece lie in the window
#pragma unroll
        for (int j0 = 0; j0 < PER; j0 += 4) {
          double w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = row.weight(x[j0 + j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float d = row.depth(x[j0 + j]);
            zc += x[j0 + j] >= negligible ? w[j] : 0.0;
            strict += d < window ? w[j] : 0.0;
            in |= d >= window && d < w1 ? 1u << (j0 + j) : 0u;
          }
        }
        if (in) {
          uint32_t to = atomicAdd(&sh.x_count, (uint32_t)__popc(in));
#pragma unroll
          for (int j = 0; j < PER; ++j)
            if (in >> j & 1u) {
              const uint32_t k = L::key(x[j]);
              if (to < (uint32_t)kList) found[to] = k;
              ++to;
              wlo = min(wlo, k);
              whi = max(whi, k);
            }
        }
      });
      wlo = __reduce_min_sync(0xffffffffu, wlo);
      whi = __reduce_max_sync(0xffffffffu, whi);
      if (lane == 0) atomicMin(&sh.x_min, wlo), atomicMax(&sh.x_top, whi);
      zc = block_sum(zc, sh.scan);
      const double above = block_sum(strict, sh.scan);
      if (tid == 0) sh.x_mass = zc, sh.x_above = above;
      cluster_sync();
      const uint32_t most = __reduce_max_sync(0xffffffffu, each_u32(&sh.x_count, nc, 0u));
      const double target = p * sum_f64(&sh.x_mass, nc), start = sum_f64(&sh.x_above, nc);
      wlo = __reduce_min_sync(0xffffffffu, each_u32(&sh.x_min, nc, kAll));
      whi = __reduce_max_sync(0xffffffffu, each_u32(&sh.x_top, nc, 0u));
      if (most > 0 && start <= target) {
        const auto c = most <= (uint32_t)kList ? row.narrow(found, (int)sh.x_count, wlo, whi, start, target)
                                               : row.template select<false, false>(wlo, whi, start, target, 0u, 0.0);
        if (c.key > wlo || c.base + c.mass > target) {  // the cut is not below the window
          cut = L::of_key(c.key);
          const double w = row.weight(cut), all = rint(c.mass / w), more = floor((target - c.base) / w) + 1.0;
          ties = (uint32_t)(more < all ? more : all);
          digits = false, summed = true;
        }
      }
    }
  }
  if (digits) {
    cluster_sync();  // the bins take what others may still read
    // a cut below T's values (a high temperature) must not become the key of -inf, whose
    // tokens would then be counted among the first ranks
    uint32_t klo = L::key(fmaxf(cut, L::kLowest)), alone = 0;
    const uint32_t khi = L::key(xmax);
    double alone_w = 0.0;
    if (klo > khi) klo = khi;
    if (cut_k) {
      const auto c = row.template select<true, false>(klo, khi, 0.0, (double)(top_k - 1), 0u, 0.0);
      cut = L::of_key(c.key);
      const double keep = (double)top_k - c.base;  // of c.mass ties
      ties = (uint32_t)(keep < c.mass ? keep : c.mass);
      klo = alone = c.key;
      alone_w = (double)ties * row.weight(cut);
    }
    if (cut_p) {
      const auto c = row.template select<false, true>(klo, khi, 0.0, p, alone, alone_w);
      cut = L::of_key(c.key);
      const double w = row.weight(cut), all = rint(c.mass / w), more = floor((c.target - c.base) / w) + 1.0;
      ties = (uint32_t)(more < all ? more : all);
    }
  }
  if (min_p > 0.0f && lowest > cut) cut = lowest, ties = kAll, summed = false;

  // kept weight above the cut and ties at it, per segment; where the weight above a window
  // is summed already, what lies between it and the cut is added
  const double w_tie = row.weight(cut);
  uint32_t tied = 0;
  if (summed) {
    row.pieces(s0, s1, PER, cut, [&](const float (&x)[PER], int) {
      uint32_t in = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const bool under = row.depth(x[j]) >= window;
        in |= under && x[j] > cut ? 1u << j : 0u;
        tied += under && x[j] == cut ? 1u : 0u;
      }
      if (in)
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (in >> j & 1u) strict += row.weight(x[j]);
    });
  } else {
    strict = 0.0;
    row.pieces(s0, s1, PER, cut, [&](const float (&x)[PER], int) {
#pragma unroll
      for (int j0 = 0; j0 < PER; j0 += 4) {
        double w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = row.weight(x[j0 + j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          strict += x[j0 + j] > cut ? w[j] : 0.0;
          tied += x[j0 + j] == cut ? 1u : 0u;
        }
      }
    });
  }
  // ties before each thread (in this CTA) and the CTA's sums
  uint32_t it = tied;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) it += v;
  }
  const double strict_all = block_sum(strict, sh.scan);
  if (lane == 31) sh.iscan[warp] = it;
  __syncthreads();
  uint32_t before = it - tied, tied_all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t v = sh.iscan[w];
    before += w < warp ? v : 0u;
    tied_all += v;
  }
  if (tid == 0) {
    sh.x_mass = strict_all;
    sh.x_ties = tied_all;
    sh.pick = kThreads;
  }
  cluster_sync();
  // every CTA finds the one that holds the target: the last one that starts at or before
  // it (a lane per CTA)
  double start, target;
  uint32_t owner;
  {
    const uint32_t t = each_u32(&sh.x_ties, nc, 0u);
    double mass = each_f64(&sh.x_mass, nc);
    uint32_t tb = t;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, tb, o);
      if (lane >= o) tb += v;
    }
    tb -= t;  // ties in the CTAs before
    mass += (double)(tb < ties ? min(t, ties - tb) : 0u) * w_tie;
    double incl = mass;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    double at = __shfl_up_sync(0xffffffffu, incl, 1);
    if (lane == 0) at = 0.0;
    start = __shfl_sync(0xffffffffu, at, rank);
    before += __shfl_sync(0xffffffffu, tb, rank);
    target = u * __shfl_sync(0xffffffffu, incl, nc - 1);
    owner = 31 - __clz(__ballot_sync(0xffffffffu, lane < (int)nc && mass > 0.0 && at <= target));
  }
  if (owner == rank) {
    const double local = target - start;
    const uint32_t mine = before < ties ? min(tied, ties - before) : 0u;
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
        const float x = i < a1 ? to_f32<T>(slice[i]) : -INFINITY;
        const uint32_t same = __ballot_sync(0xffffffffu, x == cut);
        double w = row.weight(x);
        w = x > cut ? w : 0.0;
        if (x == cut) w = tie + __popc(same & ((1u << lane) - 1u)) < ties ? w_tie : 0.0;
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

constexpr int64_t kPlaces = 264;
constexpr int kSmemMax = 200 * 1024;  // dynamic, beside the static struct

template <typename T>
int launch_filter(FilterArgs a, int64_t rows, cudaStream_t st) {
  constexpr int per = (kSmemMax - kAreaBytes) / (int)sizeof(T) / 8 * 8;
  // CTAs of a row: as few as leave two places an SM (by shared memory), since each has
  // its share of the work between the passes (64 rows of 151936 bf16, top-p 0.9: 63 us in
  // 4 CTAs, 75 in 5, 83 in 8), and up to 8 while all of them run at once (32 rows of
  // 151936: 39 us in 8, 48 in 5). Clusters of 8 fill 264 places.
  constexpr int two = (112 * 1024 - kAreaBytes - (int)sizeof(Shared)) / (int)sizeof(T);
  int nc = 1;
  while (nc < kMaxCluster && ((a.V + nc - 1) / nc > two || rows * (nc + 1) <= kPlaces)) ++nc;
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
    cfg.dynamicSmemBytes = kAreaBytes + chunk * sizeof(T);
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
