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
// keys (one pass over the logits). A cut (of top-k over counts, of top-p over
// masses) is found four key bits at a time: every thread adds its elements into 16
// bins of its own, the bins are summed in a fixed order over threads and CTAs, and
// the next pass looks only at the bin that holds the cut. The passes start at the
// range of keys whose weight is not negligible.

#include <atomic>

#include "common.cuh"

namespace csaq {
namespace {

constexpr int kThreads = 512;
constexpr int kBins = 16;  // one warp sums one bin
constexpr int kMaxCluster = 8;
constexpr int kTable = 256;           // 2^(j / 256)
constexpr double kNegligible = -50.0;  // exp below this is taken as 0: 2e-22 of the largest weight
static_assert(kBins * 32 == kThreads, "a warp per bin");

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
__device__ __forceinline__ uint32_t remote_u32(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}

// exp(z) for z in [kNegligible, 0]: table-driven reduction (Tang 1989): z = n ln2 / 256 + r,
// exp z = 2^(n / 256) (1 + r + .. + r^4 / 24), |r| <= 0.00136: within 4e-15 of it
__device__ __forceinline__ double exp_tab(double z, const double* tab) {
  const double t = rint(z * 369.3299304675746);  // 256 / ln 2
  const int n = (int)t;
  const double r = fma(t, -0.0027076061740622863, z);  // ln 2 / 256
  double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  p *= tab[n & (kTable - 1)];
  return __hiloint2double(__double2hiint(p) + ((n >> 8) << 20), __double2loint(p));
}

// What every CTA of the row knows; `red` is read by the other CTAs.
struct Shared {
  double tab[kTable];
  double red[2][kBins];  // this CTA's bin sums, alternating from pass to pass
  double tot[kBins];     // the row's
  double scan[kThreads / 32];
  uint32_t iscan[kThreads / 32];
  double x_mass;  // exchanged at the end
  uint32_t x_ties;
  uint32_t x_max;
  uint32_t wmax[kThreads / 32];
  int pick;
};

template <typename T>
struct Row {
  using KO = KeyOf<T>;
  using K = typename KO::K;
  const K* keys;  // the slice, in index order
  int n;
  Shared* sh;
  double* hist;  // [bin][thread]
  uint32_t rank, nc;
  int parity;
  bool top_inf;  // the largest logit is +inf: its like have weight 1, all else 0
  double xmax, inv_t;
  uint32_t kmax;

  __device__ __forceinline__ double weight(uint32_t k) const {
    if (top_inf) return k == kmax ? 1.0 : 0.0;
    const double z = ((double)KO::value(k) - xmax) * inv_t;
    return z >= kNegligible ? exp_tab(z, sh->tab) : 0.0;
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
    const uint32_t span = kmax - klo;
    const int bits = 32 - __clz(span | 1u);
    uint32_t prefix = 0;
    Cut c{klo, 0.0, 0.0, bound};
    bool first = true;
    for (int shift = (bits - 1) / 4 * 4; shift >= 0; shift -= 4) {
#pragma unroll
      for (int b = 0; b < kBins; ++b) hist[b * kThreads + threadIdx.x] = 0.0;
      auto add = [&](uint32_t k) {
        const uint32_t o = k - klo;  // keys below klo wrap around to far above the span
        if (o > span || k == alone || (!first && (o >> (shift + 4)) != prefix)) return;
        double* h = &hist[((o >> shift) & 15u) * kThreads + threadIdx.x];
        *h += COUNT ? 1.0 : weight(k);
      };
      for (int i = threadIdx.x; i < n; i += kThreads) add(keys[i]);
      if (alone_w != 0.0 && rank == 0 && threadIdx.x == 0) {
        const uint32_t o = alone - klo;
        if (o <= span && (first || (o >> (shift + 4)) == prefix)) hist[((o >> shift) & 15u) * kThreads] += alone_w;
      }
      __syncthreads();
      {
        const int b = threadIdx.x >> 5, lane = threadIdx.x & 31;
        double s = 0.0;
        for (int i = lane; i < kThreads; i += 32) s += hist[b * kThreads + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) sh->red[parity][b] = s;
      }
      cluster_sync();
      if (threadIdx.x < kBins) {
        double s = 0.0;
        for (uint32_t r = 0; r < nc; ++r) s += remote_f64(&sh->red[parity][threadIdx.x], r);
        sh->tot[threadIdx.x] = s;
      }
      __syncthreads();
      parity ^= 1;
      if (first && !COUNT) {
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
      prefix = (prefix << 4) | (uint32_t)pick;
      first = false;
      __syncthreads();  // tot is rewritten by the next pass
    }
    c.key = klo + prefix;
    return c;
  }
};

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
  double* hist = reinterpret_cast<double*>(dyn);
  K* keys = reinterpret_cast<K*>(dyn + kBins * kThreads * sizeof(double));
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
  row.keys = keys, row.n = n, row.sh = &sh, row.hist = hist, row.rank = rank, row.nc = nc, row.parity = 0;
  row.kmax = kmax;
  const float xmax = KO::value(kmax);
  row.top_inf = xmax == INFINITY;
  row.xmax = xmax;
  row.inv_t = greedy ? 1.0 : 1.0 / (double)temp;

  // the lowest key that can have weight: a little below max + kNegligible T
  uint32_t klo = kmax;
  if (!row.top_inf) {
    const double x = row.xmax + (kNegligible - 1.0) / row.inv_t;
    klo = x > -3.0e38 ? KO::key(from_f32<T>((float)(x - fabs(x) * 0x1p-6))) : 1u;
    if (klo == 0 || klo > kmax) klo = 1u;
  }

  // the cut: keys above ckey are kept, and the first ckeep of those at it
  uint32_t ckey = klo, cties = 0xffffffffu;
  uint32_t alone = 0;
  double alone_w = 0.0;
  if (top_k > 0 && top_k < a.V) {
    const auto c = row.template select<true>(klo, (double)(top_k - 1), 0u, 0.0);
    ckey = c.key;
    const double keep = (double)top_k - c.base;  // of c.mass ties
    cties = (uint32_t)(keep < c.mass ? keep : c.mass);
    alone = ckey;
    alone_w = (double)cties * row.weight(ckey);
  }
  if (top_p < 1.0f && !greedy) {  // NaN switches it off
    const auto c = row.template select<false>(ckey, top_p > 0.0f ? (double)top_p : 0.0, alone, alone_w);
    const double w = row.weight(c.key);
    const uint32_t all = (uint32_t)rint(c.mass / w);
    const double more = floor((c.target - c.base) / w);
    ckey = c.key;
    cties = more + 1.0 < (double)all ? (uint32_t)more + 1u : all;
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
    for (int w = 0; w < kThreads / 32; ++w) s += sh.scan[w], t += sh.iscan[w];
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

constexpr int kHistBytes = kBins * kThreads * 8;
constexpr int kSmemMax = 200 * 1024;  // dynamic, beside the static struct

template <typename T>
int launch_filter(FilterArgs a, int64_t rows, cudaStream_t st) {
  constexpr int per = (kSmemMax - kHistBytes) / (int)sizeof(typename KeyOf<T>::K) / 8 * 8;
  // CTAs of a row: as many as its keys need, and up to 8 while the rows alone
  // leave SMs idle
  int nc = 1;
  while (nc < kMaxCluster && ((a.V + nc - 1) / nc > per - 8 || rows * nc * 2 <= 148)) nc *= 2;
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
    cfg.dynamicSmemBytes = kHistBytes + chunk * sizeof(typename KeyOf<T>::K);
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
