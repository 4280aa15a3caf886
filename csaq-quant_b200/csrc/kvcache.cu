// Quantised KV cache: writing it (with the rotary embedding), reading it back,
// and decode attention that reads the codes directly.
//
// Storage of one cache (include/csaq_b200.h, csaq_kvq_cache), per layer:
//   codes  (B, Hkv, Lmax, D * bits / 8) bytes; 4-bit: even element in the low nibble
//   params (B, Hkv, Lmax, D / G) words; upper half the bf16 scale s, lower half
//          the fp16 bits of 1024 + z (0x6400 | z)
// and the value of an element is s * (code - z). The scale is a bf16 so that a
// word holds both, and it is rounded up before the codes are made: the top code
// then never clips and nothing is lost by the short scale. s * (code - z) has
// at most 8 + 9 significant bits, so it is exact in fp32. The lower half is, as
// it stands, the fp16 operand that turns a code placed in the mantissa of
// 1024.0 into code - z by one subtraction.

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <type_traits>

#include "common.cuh"

namespace csaq {
namespace {

constexpr int kMaxDev = 64;
constexpr uint32_t kZeroWord = 0x6400u;  // scale 0, zero point 0

__device__ __forceinline__ float word_scale(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float word_zero(uint32_t w) {
  return __half2float(__ushort_as_half((unsigned short)w)) - 1024.0f;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ── writing ─────────────────────────────────────────────────────────────────
// One quantisation group: s = bf16_up((max(x, 0) - min(x, 0)) / n), z = rint(-min / s),
// code = clamp(rint(x / s) + z, 0, n), every operation one fp32 rounding (no
// contraction), so that the codes are a definition and not a tolerance: values
// of 16-bit types meet the borders between codes exactly, and a correctly
// rounded quotient of them never crosses one. Zero is always representable. A
// group with a NaN or an infinity gets a NaN scale: all its values read back as
// NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// lo and hi are the extrema with zero, NaN when an element is one
template <int BITS>
__device__ __forceinline__ uint32_t group_word(float lo, float hi) {
  constexpr float n = (float)((1 << BITS) - 1);
  const float span = __fsub_rn(hi, lo);
  if (!(-lo <= FLT_MAX && hi <= FLT_MAX)) return 0x7fc00000u | kZeroWord;
  // a span beyond fp32 is taken in halves (exact at that size)
  const float s32 = span <= 3.4e38f ? __fdiv_rn(span, n) : __fdiv_rn(__fsub_rn(0.5f * hi, 0.5f * lo), 0.5f * n);
  if (!(span > 0.0f)) return kZeroWord;
  uint32_t bits = (__float_as_uint(s32) + 0xffffu) & 0xffff0000u;
  bits = bits < 0x00800000u ? 0x00800000u : bits;
  const float z = fminf(fmaxf(rintf(__fdiv_rn(-lo, __uint_as_float(bits))), 0.0f), n);
  return bits | (0x6400u + (uint32_t)z);
}

template <int BITS>
__device__ __forceinline__ uint32_t code_of(float x, float s, float z) {
  constexpr float n = (float)((1 << BITS) - 1);
  const float c = fminf(fmaxf(__fadd_rn(rintf(__fdiv_rn(x, s)), z), 0.0f), n);
  return (uint32_t)c;
}

struct WriteArgs {
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const int32_t* pos0;
  int64_t M;
  int S, Hq, Hkv;
  const float *cos_t, *sin_t;
  int n_rope;  // rows of the tables
  void* q_out;
  uint8_t *k_codes, *v_codes;
  uint32_t *k_params, *v_params;
  int Lmax;
};

// Codes of eight elements into 8 or 4 bytes. The division that defines a code costs some
// ten instructions, and a product with 1 / s, rounded, lies within 2^8 * (2^-23 + 2^-24)
// of the rounded quotient (|x / s| <= 255), so that both round to the same integer unless
// the product lies that near a half: only then (or when it is no number) do the eight
// divide. Below z nothing clips (rint(lo / s) = -z), above n it may by one.
template <int BITS>
__device__ __forceinline__ void store_half(uint8_t* dst, const float* x, float s, float inv, float z) {
  constexpr int n = (1 << BITS) - 1;
  constexpr float magic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer, ties to even
  const int base = __float_as_int(magic) - (int)z;
  int c[8];
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = __fmul_rn(x[i], inv), t = __fadd_rn(q, magic), d = fabsf(__fsub_rn(q, __fsub_rn(t, magic)));
    off = max_nan(off, d);
    c[i] = min(__float_as_int(t) - base, n);
  }
  if (!(off <= 0.5f - 1.0f / 8192.0f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = (int)code_of<BITS>(x[i], s, z);
  }
  if constexpr (BITS == 8) {
    uint2 w;
    w.x = c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24);
    w.y = c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24);
    *reinterpret_cast<uint2*>(dst) = w;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= c[i] << (4 * i);
    *reinterpret_cast<uint32_t*>(dst) = w;
  }
}

__device__ __forceinline__ void load8f(const float* p, float* out) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  out[0] = a.x; out[1] = a.y; out[2] = a.z; out[3] = a.w;
  out[4] = b.x; out[5] = b.y; out[6] = b.z; out[7] = b.w;
}

// D / 16 neighbouring threads take a head of a token: each holds elements i0..i0+7 and
// D/2+i0..D/2+i0+7, so that every rotation is its own and a group's minimum and maximum
// take log2(D / 16) shuffles. A warp holds 512 / D neighbouring tokens, whose table rows
// (four times a head's own bytes) stay in its registers while it walks over heads, one in
// every 8 * gridDim.y, so that each warp gets its share of queries, which are cheap, and
// of keys and values. The next kRing heads are on their way into shared memory meanwhile;
// each thread reads what it copied itself.
// Bound by HBM for a prompt and by latency for a decode step. 16 x 2048 tokens of 32 + 2 x 8
// heads of 128 (711 MB with 4-bit codes): 131 us, 5.4 TB/s; with the division done for every
// code 153 us. 16 tokens: 3.1 us.
constexpr int kRing = 4, kWriteBlocks = 3;
template <typename T, int BITS, int D, int G>
__global__ void __launch_bounds__(256, kWriteBlocks) kvq_write_kernel(const WriteArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint4 ring[kRing][2][256];
  constexpr int half = D / 2, TPH = D / 16, TB = 32 / TPH;
  const int nq = a.q ? a.Hq : 0, heads = nq + 2 * a.Hkv;
  const int h0 = blockIdx.y * 8 + threadIdx.x / 32, step = gridDim.y * 8;
  if (h0 >= heads) return;  // a whole warp
  const uint32_t m0 = blockIdx.x * TB + threadIdx.x % 32 / TPH;
  const bool live = m0 < (uint32_t)a.M;
  const int64_t m = live ? m0 : 0;
  const int i0 = (threadIdx.x % TPH) * 8;
  const int b = (int)((uint32_t)m / (uint32_t)a.S);
  const int64_t pos = (int64_t)a.pos0[b] + (m - (int64_t)b * a.S);
  auto load = [&](int hh, int slot) {
    if (live && hh < heads) {
      const T* src = hh < nq ? reinterpret_cast<const T*>(a.q) + m * a.ldq + (int64_t)hh * D
                             : (hh < nq + a.Hkv ? reinterpret_cast<const T*>(a.k) + m * a.ldk + (int64_t)(hh - nq) * D
                                                : reinterpret_cast<const T*>(a.v) + m * a.ldv + (int64_t)(hh - nq - a.Hkv) * D);
      cp16(smem_addr(&ring[slot][0][threadIdx.x]), src + i0);
      cp16(smem_addr(&ring[slot][1][threadIdx.x]), src + i0 + half);
    }
    cp_commit();
  };
#pragma unroll
  for (int d = 0; d < kRing; ++d) load(h0 + d * step, d);
  // a position outside the cache or the tables: its keys and values are not
  // stored and its query is passed on unrotated
  const bool in_table = !a.cos_t || (pos >= 0 && pos < a.n_rope);
  const bool keep = live && pos >= 0 && pos < a.Lmax && in_table;
  const bool turns = a.cos_t != nullptr && live && in_table && h0 < nq + a.Hkv;
  float ca[8], sa[8], cb[8], sb[8];
  if (turns) {
    load8f(a.cos_t + pos * D + i0, ca);
    load8f(a.sin_t + pos * D + i0, sa);
    load8f(a.cos_t + pos * D + i0 + half, cb);
    load8f(a.sin_t + pos * D + i0 + half, sb);
  }
  int slot = 0;
#pragma unroll 1
  for (int hh = h0; hh < heads; hh += step) {  // one head for the whole warp: its shuffles are complete
    cp_wait<kRing - 1>();
    // a thread reads back what it copied itself (zeros' place for tokens that are none)
    const uint4 u = ring[slot][0][threadIdx.x], w = ring[slot][1][threadIdx.x];
    const bool is_q = hh < nq, is_v = hh >= nq + a.Hkv;
    float lo[8], hi[8];
    const T* ue = reinterpret_cast<const T*>(&u);
    const T* we = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = to_f32<T>(ue[i]), hi[i] = to_f32<T>(we[i]);
    __syncwarp();
    load(hh + kRing * step, slot);
    slot = slot + 1 < kRing ? slot + 1 : 0;
    if (turns && !is_v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x0 = lo[i], x1 = hi[i];
        lo[i] = __fsub_rn(__fmul_rn(x0, ca[i]), __fmul_rn(x1, sa[i]));
        hi[i] = __fadd_rn(__fmul_rn(x1, cb[i]), __fmul_rn(x0, sb[i]));
      }
    }
    if (is_q) {
      if (!live) continue;
      uint4 x, y;
      T* xe = reinterpret_cast<T*>(&x);
      T* ye = reinterpret_cast<T*>(&y);
#pragma unroll
      for (int i = 0; i < 8; ++i) xe[i] = from_f32<T>(lo[i]), ye[i] = from_f32<T>(hi[i]);
      T* dst = reinterpret_cast<T*>(a.q_out) + (m * a.Hq + hh) * D;
      *reinterpret_cast<uint4*>(dst + i0) = x;
      *reinterpret_cast<uint4*>(dst + i0 + half) = y;
      continue;
    }
    float mn0 = 0.0f, mx0 = 0.0f, mn1 = 0.0f, mx1 = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mn0 = min_nan(mn0, lo[i]), mx0 = max_nan(mx0, lo[i]);
      mn1 = min_nan(mn1, hi[i]), mx1 = max_nan(mx1, hi[i]);
    }
    if constexpr (G == D) mn0 = min_nan(mn0, mn1), mx0 = max_nan(mx0, mx1);
#pragma unroll
    for (int o = 1; o < TPH; o <<= 1) {
      mn0 = min_nan(mn0, __shfl_xor_sync(0xffffffffu, mn0, o));
      mx0 = max_nan(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
      if constexpr (G != D) {
        mn1 = min_nan(mn1, __shfl_xor_sync(0xffffffffu, mn1, o));
        mx1 = max_nan(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
      }
    }
    if (!keep) continue;
    constexpr int ROWB = D * BITS / 8, NG = D / G;
    const int hk = is_v ? hh - nq - a.Hkv : hh - nq;
    const int64_t row = ((int64_t)b * a.Hkv + hk) * a.Lmax + pos;
    uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + row * ROWB;
    uint32_t* params = (is_v ? a.v_params : a.k_params) + row * NG;
    const uint32_t w0 = group_word<BITS>(mn0, mx0);
    const uint32_t w1 = G == D ? w0 : group_word<BITS>(mn1, mx1);
    // a group of zeros has scale 0 and may divide by anything
    const float s0 = word_scale(w0) != 0.0f ? word_scale(w0) : 1.0f;
    const float s1 = word_scale(w1) != 0.0f ? word_scale(w1) : 1.0f;
    store_half<BITS>(codes + i0 * BITS / 8, lo, s0, __frcp_rn(s0), (float)((w0 & 0xffffu) - kZeroWord));
    store_half<BITS>(codes + (i0 + half) * BITS / 8, hi, s1, __frcp_rn(s1), (float)((w1 & 0xffffu) - kZeroWord));
    if (i0 == 0) {
      params[0] = w0;
      if constexpr (G != D) params[1] = w1;
    }
  }
}

// ── reading back ────────────────────────────────────────────────────────────
// A thread turns 8 codes into 8 values, one 16-byte store of 16-bit values, so that a
// warp writes 512 bytes in a row; kReadUnits of them in flight. Positions
// [start, start + n) of every head; blockIdx.y strides over the (sequence, head) pairs
// and blockIdx.z picks keys or values. Bound by HBM, three quarters of it writes:
// 8 x 8 heads x 32768 positions of 128, 4-bit to fp16: 205 us, 6.7 TB/s (288 us with
// one unit of 16 a thread).
constexpr int kReadUnits = 4;
template <typename T, int BITS, int D, int G>
__global__ void __launch_bounds__(256) kvq_read_kernel(const uint8_t* __restrict__ k_codes,
                                                       const uint32_t* __restrict__ k_params,
                                                       const uint8_t* __restrict__ v_codes,
                                                       const uint32_t* __restrict__ v_params, int64_t heads, int64_t Lmax,
                                                       int64_t start, int64_t n, T* __restrict__ k_out,
                                                       T* __restrict__ v_out) {
  pdl_wait();
  pdl_trigger();
  constexpr int NG = D / G, PER = D / 8;  // units of a position
  const bool is_v = blockIdx.z != 0 || !k_out;
  const uint8_t* codes = is_v ? v_codes : k_codes;
  const uint32_t* params = is_v ? v_params : k_params;
  T* out = is_v ? v_out : k_out;
  const int64_t units = n * PER, i0 = (int64_t)blockIdx.x * (256 * kReadUnits) + threadIdx.x;
  for (int64_t bh = blockIdx.y; bh < heads; bh += gridDim.y) {
    const int64_t row = bh * Lmax + start;  // of the first position
    const uint8_t* from = codes + row * (D * BITS / 8);
    const uint32_t* words = params + row * NG;
    T* to = out + bh * n * D;
    uint2 c[kReadUnits];
    uint32_t w[kReadUnits];
#pragma unroll
    for (int u = 0; u < kReadUnits; ++u) {
      const int64_t i = i0 + u * 256;
      if (i < units) {
        if constexpr (BITS == 8)
          c[u] = __ldcs(reinterpret_cast<const uint2*>(from) + i);
        else
          c[u].x = __ldcs(reinterpret_cast<const uint32_t*>(from) + i);
        w[u] = words[i * 8 / G];
      }
    }
#pragma unroll
    for (int u = 0; u < kReadUnits; ++u) {
      const int64_t i = i0 + u * 256;
      if (i >= units) continue;
      const float s = word_scale(w[u]), z = word_zero(w[u]);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // a code in the mantissa of 2^23: subtracting 2^23 + z gives code - z, exact
        const uint32_t b = BITS == 8 ? prmt(j < 4 ? c[u].x : c[u].y, 0x4b000000u, 0x7550 + (j & 3))
                                     : (c[u].x >> (4 * j) & 15u) | 0x4b000000u;
        x[j] = (__uint_as_float(b) - (8388608.0f + z)) * s;
      }
      if constexpr (sizeof(T) == 4) {
        float4* dst = reinterpret_cast<float4*>(to + i * 8);
        __stcs(dst, make_float4(x[0], x[1], x[2], x[3]));
        __stcs(dst + 1, make_float4(x[4], x[5], x[6], x[7]));
      } else {
        uint4 v;
        T* e = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(x[j]);
        __stcs(reinterpret_cast<uint4*>(to + i * 8), v);
      }
    }
  }
}

// ── attention ───────────────────────────────────────────────────────────────
// Token (b, s) attends keys 0 .. pos0[b] + s. With codes c, zero points z and
// scales s, a score is s_k (q . c_k - z_k sum q) and an output sum_j (p_j s_j)(c_j - z_j):
// the scales leave the products, which run on the tensor cores over small integers in
// fp16, exact, with fp32 sums. They are mma.sync m16n8k16: a key meets at most 24
// query rows here, which keeps the tensor pipe under a quarter busy, and the codes go
// from shared memory through registers straight into operands, where tcgen05 would
// want them written back first. Keys take the M side of S^T = K q^T and head elements
// the M side of O^T = V^T P^T, so that 8 query rows fill an instruction. q enters as
// fp16 after a power of two per row brings its largest magnitude to [2^14, 2^15): exact
// for fp16 and bf16 q, except that elements below 2^-27 of the row's largest lose bits,
// under 2^-35 of it. Codes of K need one byte permute or AND per pair: as they stand
// they are fp16 subnormals c 2^-24, and z goes into the sum; those of V take the
// subtraction, since sums over many keys would lose what a common offset cancels.
//
// A warp takes pairs of 16-key tiles through a ring of its own (16-byte asynchronous
// copies; no barrier in the loop) and keeps its own softmax state. A CTA's 4 warps
// join theirs in warp order, then its chunk meets the others in chunk order. Tiles,
// chunks and joining order depend on key indices and on B Hkv, Lmax and the bits alone: a token's
// result does not depend on how many tokens share its step.
//
// Bound by HBM for 8 bits (4 x 8 heads x 65536 keys of 128: 94 us, 0.90 of the measured
// copy rate). 4 bits (8 x 8 x 65536: 124 us, 0.75 of it) are half the bytes with the same
// operands to build: about 340 instructions for 16 keys, 77 us if every issue slot were
// used, and two CTAs an SM leave half of them empty. The smallest calls are one chain of
// latencies (1 x 8 heads x 517 keys: 4.9 us). Many rows are short of registers and of CTAs
// (4 x 8 heads x 4101 keys, 20 rows: 19 us; of equal lengths of 2200: 17). Unequal lengths
// cost one query row a KV head a third (16 x 16 heads of 64 in 4 bits, up to 6001 keys: 30
// us; of equal lengths of 3190, as many keys in all: 20).
constexpr int kWarps = 4;
constexpr int kTile = 16;
constexpr int kStep = kWarps * 2 * kTile;  // keys that a CTA's warps take in turn
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHead = 7.0f;  // exponent of the largest weight when it sets the reference (see the state's comment)

struct AttnArgs {
  const void* q;
  int64_t ldq;
  const uint8_t *k_codes, *v_codes;
  const uint32_t *k_params, *v_params;
  const int32_t* pos0;
  int S, Hq, Hkv, Lmax, chunk;
  float scale;
  float* part;
  void* out;
  int64_t ldo;
  int bf16;
};

// two neighbouring head elements of the output, normalised; a row that sees no key is 0
__device__ __forceinline__ void store_pair(const AttnArgs& a, int64_t at, float2 v, float L) {
  const float inv = L != 0.0f ? 1.0f / L : 0.0f;
  v.x *= inv, v.y *= inv;
  if (a.bf16)
    *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<__nv_bfloat16*>(a.out) + at) = __floats2bfloat162_rn(v.x, v.y);
  else
    *reinterpret_cast<__half2*>(reinterpret_cast<__half*>(a.out) + at) = __floats2half2_rn(v.x, v.y);
}

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma16816_zero(float* c, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __half2 r = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {  // NaN only from two of them
  const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float half_of(uint32_t a, int j) {
  return __half2float(__ushort_as_half((unsigned short)(j ? a >> 16 : a)));
}
// either half above 2^15
__device__ __forceinline__ bool any_above(uint32_t a) {
  return !__hble2(*reinterpret_cast<__half2*>(&a), __floats2half2_rn(32768.0f, 32768.0f));
}
// 64 + z from 1024 + z (both halves), for nibbles read four bits up in the mantissa
__device__ __forceinline__ uint32_t zero_high(uint32_t z) { return sub2(z, 0x63806380u); }  // 960

template <int BITS, int D, int G, int NT>
struct Attn {
  static constexpr int ROWB = D * BITS / 8;       // code bytes of a key
  static constexpr int NG = D / G, NB = D / 64;   // parameter groups, 64-element blocks
  static constexpr int BPG = G / 64;              // blocks of a group
  // Tiles of a stage: two where a tile's bytes are few and the registers hold them, for
  // two independent chains of work and one vote
  static constexpr int SUB = NT == 1 && (BITS == 4 || D == 64) ? 2 : 1;
  static constexpr int KEYS = kTile * SUB;        // of a stage
  static constexpr int KV = KEYS * ROWB;          // code bytes of its keys (or values)
  static constexpr int PW = KEYS * NG;            // parameter words of its keys (or values)
  static constexpr int STAGE = 2 * KV + 8 * PW;   // keys, values, then their parameters
  static constexpr bool QSMEM = NT > 1;           // query operands reread from shared memory
  static constexpr int QBYTES = QSMEM ? kWarps * NB * 4 * NT * 256 : 0;  // of all warps: [step][n-tile][lane]
  // CTAs per SM by registers: the outputs of a thread take 16 D / 64 NT of them
  static constexpr int CTAS = NT == 1 ? 4 : (NT == 2 ? (D == 64 ? 4 : 3) : 2);
  // ring depth: what CTAS of them leave of the SM's shared memory, 8 stages at most
  static constexpr int FIT = (212 * 1024 / CTAS - QBYTES) / (kWarps * STAGE);
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  static constexpr int RING = kWarps * STAGES * STAGE;
  static constexpr int STATE = 8 * NT * (D + 2) * 4;  // of a warp or a CTA: [row][o .., m, l]
  static constexpr int JOIN = (kWarps + 1) * STATE;
  static constexpr int SMEM = (RING > JOIN ? RING : JOIN) + QBYTES;
  static_assert(STAGES >= 2, "one stage is read while the next arrives");
  // 16-byte pieces of a row are stored at piece ^ swizzle: the threads that read
  // together then meet all banks (two rows of 64 bytes already do for keys). The
  // swizzle of keys 2t, 2t + 1, 2t + 8 and 2t + 9 is one, and so is that of g and g + 8.
  static constexpr int swz_k(int key) { return ROWB == 128 ? (key & 1) << 2 : (ROWB == 64 ? key & 2 : 0); }
  static constexpr int swz_v(int key) { return ROWB == 128 ? key & 6 : (ROWB == 64 ? (key & 6) >> 1 : 0); }
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 ld_cluster(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts64(uint32_t a, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
// parameter words of one key: w[group]
template <int NG>
__device__ __forceinline__ void params1(uint32_t a, uint32_t* w) {
  if constexpr (NG == 1) {
    w[0] = lds32(a);
  } else {
    const uint2 v = lds64(a);
    w[0] = v.x, w[1] = v.y;
  }
}
// parameter words of two neighbouring keys
template <int NG>
__device__ __forceinline__ void params2(uint32_t a, uint32_t* w, uint32_t* x) {
  if constexpr (NG == 1) {
    const uint2 v = lds64(a);
    w[0] = v.x, x[0] = v.y;
  } else {
    const uint4 v = lds128(a);
    w[0] = v.x, w[1] = v.y, x[0] = v.z, x[1] = v.w;
  }
}

// fp16 operand registers of eight (4-bit) or four (8-bit) codes in `w`: for 8 bits
// {(0,1), (2,3)}, for 4 bits {(0,4), (1,5), (2,6), (3,7)}.
// raw8 / raw4: the codes as fp16 subnormals, c 2^-24, and for the odd registers of
// raw4 16 c 2^-24 (four bits up; the other operand carries the 1/16).
__device__ __forceinline__ void raw8(uint32_t w, uint32_t* r) {
  r[0] = prmt(w, 0u, 0x4140);
  r[1] = prmt(w, 0u, 0x4342);
}
__device__ __forceinline__ void raw4(uint32_t w, uint32_t* r) {
  const uint32_t x = w >> 8;
  r[0] = w & 0x000f000fu;
  r[1] = w & 0x00f000f0u;
  r[2] = x & 0x000f000fu;
  r[3] = x & 0x00f000f0u;
}
// codes8 / codes4: minus the zero point, exact small integers
__device__ __forceinline__ void codes8(uint32_t w, uint32_t z, uint32_t* r) {
  r[0] = sub2(prmt(w, 0x64646464u, 0x4140), z);
  r[1] = sub2(prmt(w, 0x64646464u, 0x4342), z);
}
__device__ __forceinline__ void codes4(uint32_t w, uint32_t z, uint32_t zh, uint32_t* r) {
  const uint32_t x = w >> 8;
  r[0] = sub2((w & 0x000f000fu) | 0x64006400u, z);
  r[1] = sub2((w & 0x00f000f0u) | 0x54005400u, zh);
  r[2] = sub2((x & 0x000f000fu) | 0x64006400u, z);
  r[3] = sub2((x & 0x00f000f0u) | 0x54005400u, zh);
}

// One warp's work on the keys of one KV head for 8 NT query rows.
template <int BITS, int D, int G, int NT>
struct WarpAttn {
  using C = Attn<BITS, D, G, NT>;
  static constexpr int NB = C::NB, NG = C::NG, ROWB = C::ROWB;
  static constexpr int RAW = D / 32;  // 16-byte pieces of a query row that a lane holds: 16 elements per block
  // 16-byte pieces: of a row of codes, of a stage's codes per lane, of a stage's parameters (keys' or values')
  static constexpr int CPR = ROWB / 16, PIECES = C::KEYS * CPR / 32, PP = C::PW / 4;
  static_assert(PIECES >= 1 && 2 * PP <= 32, "a stage's pieces are shared out to a warp");
  int lane, g, t;
  uint32_t ring, in_stage, out_stage;  // the warp's stages: first, next to fill, next to read
  const uint8_t *src_k, *src_v;        // what is copied next
  const uint32_t* src_p;
  uint32_t to_k, to_v;                 // lane offsets of its first pieces in a stage
  uint32_t qfrag;
  uint32_t at_k[NB], at_v[NB];  // lane offsets in a stage: codes of key g and value codes of key 2t, per block
  uint32_t qf[C::QSMEM ? 1 : NB * 4][2];
  float mul[NT][2];       // softmax scale, log2 e and the powers of two of rows 2t, 2t + 1
  float qsum[NT][NG][2];  // the sums of their elements per group, 2^-24 of them
  // The state of a row: a reference m, l = sum_j 2^(s_j - m), o = sum_j 2^(s_j - m) s_vj (c_j - z_j).
  // The weights 2^(s_j - m) s_vj are rounded to fp16 for the product: 2^-11 relative
  // each, below the output's own rounding for bf16 and the size of it for fp16. So
  // that they use fp16's range whatever the scale of V, m follows the largest
  // s_j + log2 s_vj: that weight is 2^kHead, and m moves only when a weight exceeds
  // 2^15 (fp16 holds 65504). Weights keep their full precision down to 2^-21 of the
  // largest and vanish below 2^-32 of it, which a million of them do not make up. m
  // starts at the lowest number: the first score exceeds it by far, and a masked one
  // (-inf) still weighs 0.
  float m[NT][2], l[NT][2], o[NT][NB * 4][4];

  __device__ __forceinline__ void setup(uint8_t* smem, int warp) {
    lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    ring = in_stage = out_stage = smem_addr(smem) + warp * (C::STAGES * C::STAGE);
    to_k = lane / CPR * ROWB + (((lane % CPR) ^ C::swz_k(lane / CPR)) * 16);
    to_v = C::KV + lane / CPR * ROWB + (((lane % CPR) ^ C::swz_v(lane / CPR)) * 16);
    qfrag = smem_addr(smem) + (C::SMEM - C::QBYTES) + warp * (C::QBYTES / kWarps) + lane * 8;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if constexpr (BITS == 8) {
        at_k[nb] = g * ROWB + (((nb * 4 + t) ^ C::swz_k(g)) * 16);
        at_v[nb] = C::KV + 2 * t * ROWB + (((nb * 4 + g / 2) ^ C::swz_v(2 * t)) * 16) + (g % 2) * 8;
      } else {
        at_k[nb] = g * ROWB + (((nb * 2 + t / 2) ^ C::swz_k(g)) * 16) + (t % 2) * 8;
        at_v[nb] = C::KV + 2 * t * ROWB + (((nb * 2 + g / 4) ^ C::swz_v(2 * t)) * 16) + (g % 4) * 4;
      }
    }
  }
  __device__ __forceinline__ uint32_t after(uint32_t stage) const {
    return stage + C::STAGE == ring + C::STAGES * C::STAGE ? ring : stage + C::STAGE;
  }

  // Where the lane's 16-byte pieces of a key-block start: `row` counts keys of all heads.
  __device__ __forceinline__ void copy_from(const AttnArgs& a, int64_t row) {
    src_k = a.k_codes + row * ROWB + lane * 16;
    src_v = a.v_codes + row * ROWB + lane * 16;
    src_p = (lane < PP ? a.k_params + lane * 4 : a.v_params + (lane - PP) * 4) + row * NG;
  }
  // Copies of the next stage, of which `left` keys exist, into the one that was read
  // last; then on by `step` keys. Piece j of a lane lies 32 / CPR keys behind piece
  // j - 1; at 8 pieces a row the swizzle of the values flips with it.
  __device__ __forceinline__ void copy_stage(int left, int step) {
    const uint32_t k = in_stage + to_k, v = in_stage + to_v;
    if (left >= C::KEYS) {
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        cp16(k + j * 512, src_k + j * 512);
        cp16((CPR == 8 && j % 2 ? v ^ 64u : v) + j * 512, src_v + j * 512);
      }
      if (lane < 2 * PP) cp16(in_stage + 2 * C::KV + lane * 16, src_p);
    } else {
#pragma unroll
      for (int j = 0; j < PIECES; ++j)
        if (lane / CPR + j * (32 / CPR) < left) {
          cp16(k + j * 512, src_k + j * 512);
          cp16((CPR == 8 && j % 2 ? v ^ 64u : v) + j * 512, src_v + j * 512);
        }
      // a piece of parameters (4 / NG keys) lies inside the buffer when its first key does (Lmax is a multiple of 16)
      if (lane < 2 * PP && (lane % PP) * 4 / NG < left) cp16(in_stage + 2 * C::KV + lane * 16, src_p);
    }
    src_k += step * ROWB;
    src_v += step * ROWB;
    src_p += step * NG;
  }

  // The lane's elements of query row 8 nt + g: 16 t .. 16 t + 15 of every block of 64.
  __device__ __forceinline__ void fetch_q(const AttnArgs& a, int b, int h, int r0, int rows, uint4 (&raw)[NT][RAW]) const {
    const int Gq = a.Hq / a.Hkv;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int rr = r0 + min(nt * 8 + g, rows - 1), s = rr / Gq, hq = h * Gq + (rr - s * Gq);
      const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + ((int64_t)b * a.S + s) * a.ldq + (int64_t)hq * D + t * 16;
#pragma unroll
      for (int i = 0; i < RAW; ++i) raw[nt][i] = *reinterpret_cast<const uint4*>(q + (i / 2) * 64 + (i % 2) * 8);
    }
  }
  // The rows as B operands of the score product, scaled by a power of two into fp16;
  // step i of block nb holds the elements that the K operand has there.
  __device__ __forceinline__ void set_q(const AttnArgs& a, int rows, const uint4 (&raw)[NT][RAW]) {
    if constexpr (C::QSMEM) __syncwarp();  // the previous rows' operands have been read
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[RAW * 8], big = 0.0f;
#pragma unroll
      for (int i = 0; i < RAW; ++i) {
        const uint32_t w[4] = {raw[nt][i].x, raw[nt][i].y, raw[nt][i].z, raw[nt][i].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned short u = (unsigned short)(j % 2 ? w[j / 2] >> 16 : w[j / 2]);
          float v = a.bf16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
          if (nt * 8 + g >= rows) v = 0.0f;
          x[i * 8 + j] = v;
          big = fmaxf(big, fabsf(v));
        }
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int e = (int)(__float_as_uint(big) >> 23) - 127;  // floor(log2), -127 for zero and subnormals
      const int up = min(14 - e, 126);
      const float f = __uint_as_float((uint32_t)(up + 127) << 23);
      // the scores come in units of 2^-24 2^-up
      const float back = a.scale * kLog2e * 0x1p24f * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        float sum = 0.0f;
#pragma unroll
        for (int i = grp * (G / 4); i < (grp + 1) * (G / 4); ++i) sum += x[i] * (f * 0x1p-24f);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qsum[nt][grp][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
        qsum[nt][grp][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      }
      mul[nt][0] = __shfl_sync(0xffffffffu, back, 8 * t);
      mul[nt][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
      for (int st = 0; st < NB * 4; ++st) {
        const float* e16 = x + (st / 4) * 16;
        const int i = st % 4, at = BITS == 8 ? 4 * i : 8 * (i / 2) + 2 * (i % 2);
        uint32_t f0, f1;
        if constexpr (BITS == 8) {
          f0 = pack2(e16[at] * f, e16[at + 1] * f);
          f1 = pack2(e16[at + 2] * f, e16[at + 3] * f);
        } else {
          f0 = pack2(e16[at] * f, e16[at + 4] * f);
          f1 = pack2(e16[at + 1] * (f * 0.0625f), e16[at + 5] * (f * 0.0625f));
        }
        if constexpr (C::QSMEM)
          sts64(qfrag + (st * NT + nt) * 256, f0, f1);
        else
          qf[st][0] = f0, qf[st][1] = f1;
      }
    }
    if constexpr (C::QSMEM) __syncwarp();
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -FLT_MAX;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < NB * 4; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
    }
  }
  // l of rows 2t, 2t + 1 over all lanes
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
      }
  }
  // o of row 8 nt + 2t + j: elements at(i), at(i) + 1 for i < 4 NB
  __device__ __forceinline__ int at(int i) const { return (i / 4) * 64 + g * 8 + (i % 4) * 2; }

  // Weights of a tile of 16 keys, and what they come from.
  struct Tile {
    float sc[NT][4];          // scores without the factor `mul`, keys g and g + 8, rows 2t and 2t + 1
    uint32_t ua[NG], ub[NG];  // the values' words of keys g and g + 8
    float p[NT][4];
    uint32_t P[NG][NT][2];    // weights times the values' scales: fp16 pairs of rows 2t, 2t + 1
  };

  // Scores of tile `sub` of a stage: s_k (q . c - z sum q).
  __device__ __forceinline__ void scores(Tile& x, uint32_t stage, int sub) const {
    const uint32_t at_p = stage + 2 * C::KV + (sub * 16 + g) * NG * 4, codes = stage + sub * 16 * ROWB;
    uint32_t wa[NG], wb[NG];  // keys g and g + 8
    params1<NG>(at_p, wa);
    params1<NG>(at_p + 8 * NG * 4, wb);
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      float acc[NT][4];
#pragma unroll
      for (int bb = 0; bb < C::BPG; ++bb) {
        const int nb = grp * C::BPG + bb;
        uint32_t A[4][4];
        if constexpr (BITS == 8) {
          const uint4 ca = lds128(codes + at_k[nb]), cb = lds128(codes + at_k[nb] + 8 * ROWB);
          const uint32_t xa[4] = {ca.x, ca.y, ca.z, ca.w}, xb[4] = {cb.x, cb.y, cb.z, cb.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t ra[2], rb[2];
            raw8(xa[i], ra);
            raw8(xb[i], rb);
            A[i][0] = ra[0], A[i][1] = rb[0], A[i][2] = ra[1], A[i][3] = rb[1];
          }
        } else {
          const uint2 ca = lds64(codes + at_k[nb]), cb = lds64(codes + at_k[nb] + 8 * ROWB);
          const uint32_t xa[2] = {ca.x, ca.y}, xb[2] = {cb.x, cb.y};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t ra[4], rb[4];
            raw4(xa[i], ra);
            raw4(xb[i], rb);
            A[2 * i][0] = ra[0], A[2 * i][1] = rb[0], A[2 * i][2] = ra[1], A[2 * i][3] = rb[1];
            A[2 * i + 1][0] = ra[2], A[2 * i + 1][1] = rb[2], A[2 * i + 1][2] = ra[3], A[2 * i + 1][3] = rb[3];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t B[2];
            if constexpr (C::QSMEM) {
              const uint2 f = lds64(qfrag + ((nb * 4 + i) * NT + nt) * 256);
              B[0] = f.x, B[1] = f.y;
            } else {
              B[0] = qf[nb * 4 + i][0], B[1] = qf[nb * 4 + i][1];
            }
            if (bb == 0 && i == 0)
              mma16816_zero(acc[nt], A[i], B);
            else
              mma16816(acc[nt], A[i], B);
          }
      }
      const float sa = word_scale(wa[grp]), sb = word_scale(wb[grp]);
      const float za = word_zero(wa[grp]), zb = word_zero(wb[grp]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float da = fmaf(-za, qsum[nt][grp][j], acc[nt][j]), db = fmaf(-zb, qsum[nt][grp][j], acc[nt][2 + j]);
          x.sc[nt][j] = grp == 0 ? da * sa : fmaf(da, sa, x.sc[nt][j]);
          x.sc[nt][2 + j] = grp == 0 ? db * sb : fmaf(db, sb, x.sc[nt][2 + j]);
        }
    }
    params1<NG>(at_p + C::PW * 4, x.ua);
    params1<NG>(at_p + C::PW * 4 + 8 * NG * 4, x.ub);
  }

  // The tile's weights under the current references; lo = li + their sums. seen(row)
  // keys from the tile's first on are visible (WHOLE: all). One arithmetic for whole
  // and cut tiles: a token's bits must not depend on which of them it meets.
  template <bool WHOLE, typename S>
  __device__ __forceinline__ bool masked(int nt, int i, S seen) const {
    return !WHOLE && g + (i / 2) * 8 >= seen(nt * 8 + 2 * t + i % 2);
  }
  template <bool WHOLE, typename S>
  __device__ __forceinline__ void weigh(Tile& x, const float (&li)[NT][2], float (&lo)[NT][2], S seen) const {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x.p[nt][i] = ex2(fmaf(x.sc[nt][i], mul[nt][i % 2], -m[nt][i % 2]));
        if (masked<WHOLE>(nt, i, seen)) x.p[nt][i] = 0.0f;
      }
      lo[nt][0] = li[nt][0] + (x.p[nt][0] + x.p[nt][2]);
      lo[nt][1] = li[nt][1] + (x.p[nt][1] + x.p[nt][3]);
#pragma unroll
      for (int grp = 0; grp < NG; ++grp)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float v = word_scale(k ? x.ub[grp] : x.ua[grp]);
          float w0 = x.p[nt][2 * k] * v, w1 = x.p[nt][2 * k + 1] * v;
          if (masked<WHOLE>(nt, 2 * k, seen)) w0 = 0.0f;  // a masked key's scale may be anything
          if (masked<WHOLE>(nt, 2 * k + 1, seen)) w1 = 0.0f;
          x.P[grp][nt][k] = pack2(w0, w1);
        }
    }
  }
  __device__ __forceinline__ uint32_t largest(const Tile& x, int nt) const {  // weights of rows 2t, 2t + 1
    uint32_t top = max2(x.P[0][nt][0], x.P[0][nt][1]);
#pragma unroll
    for (int grp = 1; grp < NG; ++grp) top = max2(top, max2(x.P[grp][nt][0], x.P[grp][nt][1]));
    return top;
  }
  // Weights above 2^15 call for a new reference; under scales of (nearly) 0 they say
  // nothing, and there the bound is on l. A reference only rises: many keys under scales
  // of 0 take l beyond its bound with weights of up to 2^87 each, and the scores that come
  // after them may all be far lower, or masked. 2^30 such keys make 2^117, still finite.
  static constexpr float kMost = 0x1p95f;

  // New references for the rows whose weights call for them: each by its own weights
  // alone, whatever the other rows do.
  template <bool WHOLE, typename S>
  __device__ __forceinline__ void refer(const Tile& x, const float (&lo)[NT][2], S seen) {
    // log2 of the values' scales, from -80 on: no weight 2^(s - m) exceeds 2^87 then
    float ea = 0.0f, eb = 0.0f;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) ea = fmaxf(ea, word_scale(x.ua[grp])), eb = fmaxf(eb, word_scale(x.ub[grp]));
    ea = fmaxf(lg2(ea), -80.0f);
    eb = fmaxf(lg2(eb), -80.0f);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t top = largest(x, nt);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float call = lo[nt][j] > kMost || half_of(top, j) > 0x1p15f ? 1.0f : 0.0f;
        const float sa = masked<WHOLE>(nt, j, seen) ? -INFINITY : x.sc[nt][j] * mul[nt][j] + ea;
        const float sb = masked<WHOLE>(nt, 2 + j, seen) ? -INFINITY : x.sc[nt][2 + j] * mul[nt][j] + eb;
        float high = fmaxf(sa, sb);
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          call = fmaxf(call, __shfl_xor_sync(0xffffffffu, call, k));
          high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, k));
        }
        if (call > 0.0f) {
          const float to = fmaxf(m[nt][j], high - kHead);
          const float f = ex2(m[nt][j] - to);  // 0 from the start
          m[nt][j] = to;
          l[nt][j] *= f;
#pragma unroll
          for (int i = 0; i < NB * 4; ++i) {
            o[nt][i][j] *= f;
            o[nt][i][2 + j] *= f;
          }
        }
      }
    }
  }

  // o += the tile's weighted values: keys 2t, 2t + 1, 2t + 8, 2t + 9, head elements
  // 8g .. of each block. `last` keys from the tile's first on exist.
  template <bool WHOLE>
  __device__ __forceinline__ void values(const Tile& x, uint32_t stage, int sub, int last) {
    const uint32_t at_p = stage + 2 * C::KV + C::PW * 4 + (sub * 16 + 2 * t) * NG * 4, codes = stage + sub * 16 * ROWB;
    uint32_t w0[NG], w1[NG], w2[NG], w3[NG];
    params2<NG>(at_p, w0, w1);
    params2<NG>(at_p + 8 * NG * 4, w2, w3);
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      uint32_t B[NT][2];  // the weights as B operands (a transposition of 8 keys x 8 rows)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        B[nt][0] = transpose8x8(x.P[grp][nt][0]);
        B[nt][1] = transpose8x8(x.P[grp][nt][1]);
      }
      if constexpr (!WHOLE) {  // the zero points behind the last key must be numbers
        w0[grp] = 2 * t < last ? w0[grp] : kZeroWord;
        w1[grp] = 2 * t + 1 < last ? w1[grp] : kZeroWord;
        w2[grp] = 2 * t + 8 < last ? w2[grp] : kZeroWord;
        w3[grp] = 2 * t + 9 < last ? w3[grp] : kZeroWord;
      }
      const uint32_t z01 = prmt(w0[grp], w1[grp], 0x5410), z23 = prmt(w2[grp], w3[grp], 0x5410);
      const uint32_t z01h = zero_high(z01), z23h = zero_high(z23);
#pragma unroll
      for (int bb = 0; bb < C::BPG; ++bb) {
        const int nb = grp * C::BPG + bb;
        const uint32_t vs = codes + at_v[nb];
        uint2 y0, y1, y2, y3;
        if constexpr (BITS == 8) {
          y0 = lds64(vs), y1 = lds64(vs + ROWB), y2 = lds64(vs + 8 * ROWB), y3 = lds64(vs + 9 * ROWB);
        } else {
          y0.x = lds32(vs), y1.x = lds32(vs + ROWB), y2.x = lds32(vs + 8 * ROWB), y3.x = lds32(vs + 9 * ROWB);
        }
        // two halves of the block's eight elements: E[e] = keys (2t, 2t + 1), (2t + 8, 2t + 9)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t E[4][2];
          if constexpr (BITS == 8) {
            const uint32_t x0 = hf ? y0.y : y0.x, x1 = hf ? y1.y : y1.x, x2 = hf ? y2.y : y2.x, x3 = hf ? y3.y : y3.x;
            uint32_t r[2];
            codes8(prmt(x0, x1, 0x5140), z01, r);
            E[0][0] = r[0], E[1][0] = r[1];
            codes8(prmt(x0, x1, 0x7362), z01, r);
            E[2][0] = r[0], E[3][0] = r[1];
            codes8(prmt(x2, x3, 0x5140), z23, r);
            E[0][1] = r[0], E[1][1] = r[1];
            codes8(prmt(x2, x3, 0x7362), z23, r);
            E[2][1] = r[0], E[3][1] = r[1];
          } else {
            uint32_t r[4];
            codes4(prmt(y0.x, y1.x, hf ? 0x7632 : 0x5410), z01, z01h, r);
#pragma unroll
            for (int e = 0; e < 4; ++e) E[e][0] = r[e];
            codes4(prmt(y2.x, y3.x, hf ? 0x7632 : 0x5410), z23, z23h, r);
#pragma unroll
            for (int e = 0; e < 4; ++e) E[e][1] = r[e];
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t A[4] = {E[2 * i][0], E[2 * i + 1][0], E[2 * i][1], E[2 * i + 1][1]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][nb * 4 + hf * 2 + i], A, B[nt]);
          }
        }
      }
    }
  }

  // The stage at out_stage: SUB tiles of 16 keys from key0 on. WHOLE: every key is
  // visible to every row; else visible(row) of all keys are, and none behind `last`.
  // The tiles have their effect one after the other, as if each had a stage of its own;
  // only while no row needs a new reference are they worked on together.
  template <bool WHOLE, typename V>
  __device__ __forceinline__ void stage(const int key0, const int last, V visible) {
    const uint32_t at = out_stage;
    Tile x[C::SUB];
    float lo[C::SUB][NT][2];
    bool over = false;
#pragma unroll
    for (int i = 0; i < C::SUB; ++i) scores(x[i], at, i);
#pragma unroll
    for (int i = 0; i < C::SUB; ++i) {
      weigh<WHOLE>(x[i], i == 0 ? l : lo[i > 0 ? i - 1 : 0], lo[i], [&](int r) { return visible(r) - key0 - 16 * i; });
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        over = over || any_above(largest(x[i], nt)) || fmaxf(lo[i][nt][0], lo[i][nt][1]) > kMost;
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int i = 0; i < C::SUB; ++i) {
        auto seen = [&](int r) { return visible(r) - key0 - 16 * i; };
        if (i > 0) weigh<WHOLE>(x[i], l, lo[i], seen);
        refer<WHOLE>(x[i], lo[i], seen);
        weigh<WHOLE>(x[i], l, lo[i], seen);
        set_l(lo[i]);
        values<WHOLE>(x[i], at, i, last - key0 - 16 * i);
      }
    } else {
      set_l(lo[C::SUB - 1]);
#pragma unroll
      for (int i = 0; i < C::SUB; ++i) values<WHOLE>(x[i], at, i, last - key0 - 16 * i);
    }
    in_stage = out_stage;  // read by this lane; by all when the next stage begins
    out_stage = after(out_stage);
  }
  __device__ __forceinline__ void set_l(const float (&from)[NT][2]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) l[nt][0] = from[nt][0], l[nt][1] = from[nt][1];
  }
};

// Keys visible to query row r of a sequence at p0 of which `len` keys are visible to anyone.
__device__ __forceinline__ int visible_keys(int64_t p0, int len, int r, int R, int Gq) {
  const int64_t l = p0 + min(r, R - 1) / Gq + 1;
  return (int)(l < 0 ? 0 : (l > len ? len : l));
}
__device__ __forceinline__ int length_of(const AttnArgs& a, int64_t p0) {
  const int64_t end = p0 + a.S;
  return (int)(end < 0 ? 0 : (end > a.Lmax ? a.Lmax : end));
}

// A CTA takes one chunk of a head's keys for one row block (grid: head, chunk, row
// block), its warps every fourth tile of it. The chunks of a head meet in shared
// memory when they are the CTAs of one cluster, else as partials in global memory.
template <int BITS, int D, int G, int NT>
__global__ void __launch_bounds__(kWarps * 32, Attn<BITS, D, G, NT>::CTAS) kvq_attention_kernel(const AttnArgs a) {
  using C = Attn<BITS, D, G, NT>;
  constexpr int NB = C::NB, kThreads = kWarps * 32;
  extern __shared__ __align__(128) uint8_t smem[];
  WarpAttn<BITS, D, G, NT> w;
  const int warp = threadIdx.x >> 5;
  w.setup(smem, warp);
  const int bh = blockIdx.x, b = bh / a.Hkv, h = bh - b * a.Hkv;
  const int Gq = a.Hq / a.Hkv, R = a.S * Gq;  // query heads per KV head, query rows of the head
  const int r0 = blockIdx.z * 8 * NT, rows = min(8 * NT, R - r0);
  const int chunk_at = blockIdx.y;  // the place in the cluster too, when the y extent is one
  pdl_wait();
  pdl_trigger();
  uint4 raw[NT][C::NB * 2];
  w.fetch_q(a, b, h, r0, rows, raw);
  const int64_t p0 = a.pos0[b];
  const int len = length_of(a, p0);
  const int n_act = len > a.chunk ? (len + a.chunk - 1) / a.chunk : 1;  // chunks with keys
  if (chunk_at >= n_act) return;  // a CTA that has left counts as arrived in its cluster's barriers
  const int k0 = chunk_at * a.chunk, k1 = min(len, k0 + a.chunk);
  // This warp's tiles: two neighbours from `first` on, the next two kStep keys later.
  // (Stages of one tile keep to that order.)
  const int first = k0 + warp * 2 * kTile;
  w.copy_from(a, (int64_t)bh * a.Lmax + first);
  int to_copy = first;
  auto issue = [&]() {
    if (to_copy < k1) {
      const int step = C::SUB == 2 ? kStep : ((to_copy & kTile) == 0 ? kTile : kStep - kTile);
      w.copy_stage(k1 - to_copy, step);
      to_copy += step;
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) {
    w.in_stage = w.ring + i * C::STAGE;
    issue();
  }
  w.in_stage = w.ring + (C::STAGES - 1) * C::STAGE;
  w.set_q(a, rows, raw);
  w.clear();
  auto visible = [&](int r) { return visible_keys(p0, len, r0 + r, R, Gq); };
  const int whole = min(visible(0), k1) - C::KEYS;  // stages from up to here are seen whole by every row
  int key = first;
  auto next = [&]() {
    cp_wait<C::STAGES - 2>();
    __syncwarp();  // the stage is in shared memory for every lane, and the previous one has been read
    issue();
  };
  auto step = [&]() { key += C::SUB == 2 ? kStep : ((key & kTile) == 0 ? kTile : kStep - kTile); };
  for (; key <= whole; step()) {
    next();
    w.template stage<true>(key, k1, visible);
  }
  for (; key < k1; step()) {
    next();
    w.template stage<false>(key, k1, visible);
  }
  cp_wait<0>();
  w.finish();
  __syncthreads();  // every warp has read its last tile: the ring becomes the joining buffer

  // The warps' states join in warp order into the CTA's, behind them in the buffer.
  float* join = reinterpret_cast<float*>(smem);
  float* mine = join + kWarps * (C::STATE / 4);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float* to = join + (warp * 8 * NT + nt * 8 + 2 * w.t + j) * (D + 2);
#pragma unroll
      for (int i = 0; i < NB * 4; ++i)
        *reinterpret_cast<float2*>(to + w.at(i)) = make_float2(w.o[nt][i][j], w.o[nt][i][2 + j]);
      if (w.g == 0) *reinterpret_cast<float2*>(to + D) = make_float2(w.m[nt][j], w.l[nt][j]);
    }
  __syncthreads();
  auto output = [&](int r, int d, float2 v, float L) {
    const int rr = r0 + r, s = rr / Gq, hq = h * Gq + (rr - s * Gq);
    store_pair(a, ((int64_t)b * a.S + s) * a.ldo + (int64_t)hq * D + d, v, L);
  };
  // [bh][chunk][row][D + 2]
  float* part = a.part + (((int64_t)bh * gridDim.y + chunk_at) * R + r0) * (D + 2);
  for (int e = threadIdx.x; e < rows * (D / 2); e += kThreads) {
    const int r = e / (D / 2), d = (e % (D / 2)) * 2;
    const float* from = join + r * (D + 2);
    float2 ml[kWarps];
    float top = -FLT_MAX, L = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      ml[i] = *reinterpret_cast<const float2*>(from + i * (C::STATE / 4) + D);
      top = fmaxf(top, ml[i].x);
    }
    float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float f = ex2(ml[i].x - top);
      const float2 v = *reinterpret_cast<const float2*>(from + i * (C::STATE / 4) + d);
      L = fmaf(ml[i].y, f, L);
      acc.x = fmaf(v.x, f, acc.x);
      acc.y = fmaf(v.y, f, acc.y);
    }
    if (n_act == 1) {
      output(r, d, acc, L);
    } else {
      float* to = a.part ? part + r * (D + 2) : mine + r * (D + 2);
      *reinterpret_cast<float2*>(to + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(to + D) = make_float2(top, L);
    }
  }
  if (n_act == 1 || a.part) return;
  cluster_sync();
  // The CTAs join their states in chunk order, a share of the elements each.
  const uint32_t mine_a = smem_addr(mine);
  for (int e = chunk_at * kThreads + threadIdx.x; e < rows * (D / 2); e += n_act * kThreads) {
    const int r = e / (D / 2), d = (e % (D / 2)) * 2;
    float2 ml[kMaxCluster], v[kMaxCluster];
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      const uint32_t from = cluster_addr(mine_a + r * (D + 2) * 4, c < n_act ? c : 0);
      ml[c] = ld_cluster(from + D * 4);
      v[c] = ld_cluster(from + d * 4);
    }
    float top = -FLT_MAX, L = 0.0f;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) top = fmaxf(top, c < n_act ? ml[c].x : -FLT_MAX);
    float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      if (c < n_act) {
        const float f = ex2(ml[c].x - top);
        L = fmaf(ml[c].y, f, L);
        acc.x = fmaf(v[c].x, f, acc.x);
        acc.y = fmaf(v[c].y, f, acc.y);
      }
    }
    output(r, d, acc, L);
  }
  cluster_sync();  // no CTA leaves while another reads its state
}

// The join of a head's chunks, one CTA a query row: its warps take every fourth chunk
// each, in order, and their sums meet in warp order. The chunks' weights come first,
// 32 of them a lane each, so that the loads of the sums do not wait for one another.
template <int D>
__global__ void __launch_bounds__(128) kvq_join_kernel(const AttnArgs a, int n_split) {
  __shared__ float tops[4];
  __shared__ float sums[4][D + 1];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;  // (b, h, r)
  const int Gq = a.Hq / a.Hkv, R = a.S * Gq;
  const int64_t bh = row / R;
  const int r = (int)(row - bh * R), b = (int)(bh / a.Hkv), h = (int)(bh - (int64_t)b * a.Hkv);
  const int len = length_of(a, a.pos0[b]);
  const int n_act = len > a.chunk ? (len + a.chunk - 1) / a.chunk : 1;
  if (n_act == 1) return;  // its only chunk was the output
  const float* part = a.part + (bh * n_split * R + r) * (D + 2);
  const int64_t step = (int64_t)R * (D + 2);
  float top = -FLT_MAX;
  for (int c = threadIdx.x; c < n_act; c += 128) top = fmaxf(top, __ldcg(part + c * step + D));
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  constexpr int PAIRS = D / 64;  // of elements per lane: 2 (lane + 32 i)
  float L = 0.0f;
  float2 acc[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) acc[i] = make_float2(0.0f, 0.0f);
  for (int c0 = warp; c0 < n_act; c0 += 128) {  // chunks c0, c0 + 4, .. c0 + 124
    const int nc = min(32, (n_act - c0 + 3) / 4);
    float2 ml = make_float2(-FLT_MAX, 0.0f);
    if (lane < nc) ml = __ldcg(reinterpret_cast<const float2*>(part + (c0 + 4 * lane) * step + D));
    const float f = ex2(ml.x - top);
#pragma unroll 8
    for (int c = 0; c < nc; ++c) {
      const float fc = __shfl_sync(0xffffffffu, f, c), lc = __shfl_sync(0xffffffffu, ml.y, c);
      L = fmaf(lc, fc, L);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(part + (c0 + 4 * c) * step) + lane + 32 * i);
        acc[i].x = fmaf(v.x, fc, acc[i].x);
        acc[i].y = fmaf(v.y, fc, acc[i].y);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    sums[warp][2 * (lane + 32 * i)] = acc[i].x;
    sums[warp][2 * (lane + 32 * i) + 1] = acc[i].y;
  }
  if (lane == 0) sums[warp][D] = L;
  __syncthreads();
  const int d = 2 * threadIdx.x;
  if (d >= D) return;
  float2 v = make_float2(0.0f, 0.0f);
  L = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.x += sums[i][d], v.y += sums[i][d + 1], L += sums[i][D];
  const int s = r / Gq, hq = h * Gq + r % Gq;
  store_pair(a, ((int64_t)b * a.S + s) * a.ldo + (int64_t)hq * D + d, v, L);
}

// ── host side ───────────────────────────────────────────────────────────────
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// CSAQ_OK when the cache descriptor fits heads of D elements
int check_cache(const csaq_kvq_cache* c, int64_t B, int64_t Hkv, int64_t D) {
  if (!c || !c->k_codes || !c->k_params || !c->v_codes || !c->v_params) return CSAQ_ERR_ARG;
  if (B <= 0 || Hkv <= 0 || D <= 0 || c->Lmax <= 0) return CSAQ_ERR_ARG;
  if (c->bits != 8 && c->bits != 4) return CSAQ_ERR_BITS;
  if ((D != 64 && D != 128) || c->Lmax % 16 || c->Lmax > (1 << 30)) return CSAQ_ERR_UNSUPPORTED;
  if (c->group_size != D && c->group_size != 64) return CSAQ_ERR_UNSUPPORTED;
  if (B * Hkv > INT32_MAX / 2) return CSAQ_ERR_UNSUPPORTED;
  if (!aligned16(c->k_codes) || !aligned16(c->k_params) || !aligned16(c->v_codes) || !aligned16(c->v_params))
    return CSAQ_ERR_UNSUPPORTED;
  return CSAQ_OK;
}

// f.template operator()<BITS, D, G>() for the cache's layout
template <typename F>
int by_layout(const csaq_kvq_cache* c, int64_t D, F f) {
  if (D == 64) return c->bits == 8 ? f.template run<8, 64, 64>() : f.template run<4, 64, 64>();
  if (c->group_size == 128) return c->bits == 8 ? f.template run<8, 128, 128>() : f.template run<4, 128, 128>();
  return c->bits == 8 ? f.template run<8, 128, 64>() : f.template run<4, 128, 64>();
}

struct LaunchWrite {
  const WriteArgs& a;
  int dtype;
  cudaStream_t st;
  template <int BITS, int D, int G>
  int run() const {
    const int64_t heads = (a.q ? a.Hq : 0) + 2 * (int64_t)a.Hkv;
    if (a.M > INT32_MAX || heads > 65535) return CSAQ_ERR_UNSUPPORTED;
    if (dtype == CSAQ_DT_BF16) return go<__nv_bfloat16, BITS, D, G>(heads);
    return go<__half, BITS, D, G>(heads);
  }
  template <typename T, int BITS, int D, int G>
  int go(int64_t heads) const {
    constexpr int TB = 512 / D;  // tokens of a warp
    const int64_t bx = (a.M + TB - 1) / TB, by = (heads + 7) / 8;
    // heads a warp takes: one while the CTAs fit the SMs together, up to eight when there
    // are more tokens than that (16 x 2048 tokens: 131 us with six, 152 with three)
    const int64_t each = std::max<int64_t>(1, std::min<int64_t>(8, bx * by / (148 * kWriteBlocks)));
    const dim3 grid((unsigned)bx, (unsigned)((by + each - 1) / each));
    return launch_pdl(kvq_write_kernel<T, BITS, D, G>, grid, dim3(256), 0, st, a);
  }
};

struct LaunchRead {
  const csaq_kvq_cache* c;
  int64_t heads, start, n;
  void *k_out, *v_out;
  int dtype;
  cudaStream_t st;
  template <typename T, int BITS, int D, int G>
  int go() const {
    const int64_t bx = (n * (D / 8) + 256 * kReadUnits - 1) / (256 * kReadUnits);
    if (bx > INT32_MAX) return CSAQ_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)bx, (unsigned)(heads < 65535 ? heads : 65535), k_out && v_out ? 2 : 1);
    return launch_pdl(kvq_read_kernel<T, BITS, D, G>, grid, dim3(256), 0, st, c->k_codes, c->k_params, c->v_codes,
                      c->v_params, heads, c->Lmax, start, n, (T*)k_out, (T*)v_out);
  }
  template <int BITS, int D, int G>
  int run() const {
    if (dtype == CSAQ_DT_BF16) return go<__nv_bfloat16, BITS, D, G>();
    if (dtype == CSAQ_DT_F16) return go<__half, BITS, D, G>();
    return go<float, BITS, D, G>();
  }
};

// How a cache is cut into chunks, from B * Hkv, Lmax and the bits alone (so that a step's token
// count does not move the borders). Up to 8 chunks a head are the CTAs of a cluster: as
// many as one wave takes, and of kEven keys and more up to four waves of them, which even
// out unequal lengths: 32 x 8 heads, 8-bit, of up to 8192 keys take 57 us in 6 chunks, 60
// in 8 and 67 in 2, of up to 32768 198 in 8, 211 in 6 and 245 in 2, of up to 1024 14 in 2 and
// 20 in 8. Where 8 leave SMs without a CTA and the cache is long, one wave
// of CTAs leaves partials: 1 x 8 heads x 131072 keys, 8-bit, 58 us against 117; at
// 8192 keys the second kernel costs what the wave gains (11.6 and 11.1 us). 4-bit codes,
// bound by instructions, gain from a full wave at up to 73 heads, too, once they are long:
// 4 x 8 heads x 65536 keys 69 us against 88, 7 x 8 x 32768 63 against 71, and 4 x 8 x 16384
// 26 either way; 8-bit ones lose there (4 x 8 x 65536: 102 against 98).
struct Split {
  int chunk, n;
  bool partial;
};
constexpr int64_t kSms = 148, kSlots = 4 * kSms;  // CTAs that run at once (one row block of up to 8 rows)
constexpr int64_t kEven = 1280;  // keys of a chunk that only evens out lengths
Split split_of(int64_t heads, int64_t Lmax, int bits) {
  Split s;
  s.partial = heads * kMaxCluster < kSms ? Lmax > 8192 : bits == 4 && heads * kMaxCluster < kSlots && Lmax > 16384;
  int64_t n = std::max<int64_t>(kSlots / heads, 1);
  if (!s.partial) n = std::min<int64_t>(kMaxCluster, std::max(n, std::min(4 * kSlots / heads, Lmax / kEven)));
  s.chunk = (int)(((Lmax + n - 1) / n + kStep - 1) / kStep * kStep);
  s.n = (int)((Lmax + s.chunk - 1) / s.chunk);
  return s;
}

struct LaunchAttn {
  const AttnArgs& a;
  int64_t B;
  Split split;
  cudaStream_t st;
  template <typename K>
  int ready(K kern, int smem, std::atomic<uint64_t>& done) const {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= kMaxDev)) return CSAQ_ERR_UNSUPPORTED;
    if (e == cudaSuccess && !(done.load(std::memory_order_relaxed) >> dev & 1)) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e == cudaSuccess) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    if (e == cudaSuccess) return CSAQ_OK;
    set_last_cuda_error(e);
    (void)cudaGetLastError();
    return CSAQ_ERR_CUDA;
  }
  template <int BITS, int D, int G, int NT>
  int go() const {
    using C = Attn<BITS, D, G, NT>;
    static std::atomic<uint64_t> done{0};  // devices on which the kernel's shared memory is set
    const int64_t R = (int64_t)a.S * (a.Hq / a.Hkv), nz = (R + 8 * NT - 1) / (8 * NT), heads = B * a.Hkv;
    auto kern = kvq_attention_kernel<BITS, D, G, NT>;
    if (nz > 65535 || split.n > 65535 || heads * R > INT32_MAX) return CSAQ_ERR_UNSUPPORTED;
    const int rc = ready(kern, C::SMEM, done);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)heads, (unsigned)split.n, (unsigned)nz);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
    attr[0].val.clusterDim.y = split.partial ? 1 : split.n;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
    if (e != cudaSuccess) {
      set_last_cuda_error(e);
      (void)cudaGetLastError();
      return CSAQ_ERR_CUDA;
    }
    const int lrc = launch_status();
    if (lrc || !split.partial) return lrc;
    return launch_pdl(kvq_join_kernel<D>, dim3((unsigned)(heads * R)), dim3(128), 0, st, a, split.n);
  }
  template <int BITS, int D, int G>
  int run() const {
    const int64_t R = (int64_t)a.S * (a.Hq / a.Hkv);
    // Rows of a CTA: all of them while that is 24, since each block of rows builds its
    // operands from the codes anew (16 x 8 heads x 4096 keys, 20 rows: 48 us with 24, 64 with
    // two blocks of 16, 69 with three of 8), and 16 from then on (16 x 8 x 8192, 32 rows:
    // 114 us with 16, 160 with 24, which run twice an SM).
    // Blocks of 8 when all CTAs then run at once: few CTAs wait for latency (8 heads x 4096
    // keys, 20 rows: 10.0 us with 8, 13.1 with 24; x 2048, 64 rows: 10.3 with 8, 12.0 with 16).
    if (R <= 8 || B * a.Hkv * split.n * ((R + 7) / 8) <= kSlots) return go<BITS, D, G, 1>();
    return R <= 16 || R > 24 ? go<BITS, D, G, 2>() : go<BITS, D, G, 3>();
  }
};

}  // namespace
}  // namespace csaq

using namespace csaq;

extern "C" int csaq_kvq_write(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                              const int32_t* pos0, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                              const float* cos_t, const float* sin_t, int64_t n_rope, void* q_out,
                              const csaq_kvq_cache* cache, int dtype, void* stream) {
  const int rc = check_cache(cache, B, Hkv, D);
  if (rc) return rc;
  if (!k || !v || !pos0 || S <= 0 || (q && (!q_out || Hq <= 0)) || !cos_t != !sin_t || (cos_t && n_rope <= 0))
    return CSAQ_ERR_ARG;
  if (q && !cos_t) return CSAQ_ERR_ARG;  // nothing would be done to the queries
  if (dtype != CSAQ_DT_F16 && dtype != CSAQ_DT_BF16) return CSAQ_ERR_ARG;
  if (ldk < Hkv * D || ldv < Hkv * D || (q && ldq < Hq * D)) return CSAQ_ERR_ARG;
  if (ldk % 8 || ldv % 8 || (q && ldq % 8) || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) ||
      !aligned16(cos_t) || !aligned16(sin_t))
    return CSAQ_ERR_UNSUPPORTED;
  if (S > INT32_MAX || B * S > INT32_MAX || Hq > INT32_MAX / 4 || n_rope > INT32_MAX) return CSAQ_ERR_UNSUPPORTED;
  const WriteArgs a{q,     k,     v,     ldq,           ldk,   ldv,           pos0,           B * S,
                    (int)S, (int)Hq, (int)Hkv, cos_t, sin_t, (int)n_rope,   q_out,          cache->k_codes,
                    cache->v_codes, cache->k_params, cache->v_params, (int)cache->Lmax};
  return by_layout(cache, D, LaunchWrite{a, dtype, as_stream(stream)});
}

extern "C" int csaq_kvq_read(const csaq_kvq_cache* cache, int64_t B, int64_t Hkv, int64_t D, int64_t start, int64_t n,
                             void* k_out, void* v_out, int dtype, void* stream) {
  const int rc = check_cache(cache, B, Hkv, D);
  if (rc) return rc;
  if ((!k_out && !v_out) || start < 0 || n < 0 || start > cache->Lmax || n > cache->Lmax - start) return CSAQ_ERR_ARG;
  if (dtype != CSAQ_DT_F16 && dtype != CSAQ_DT_BF16 && dtype != CSAQ_DT_F32) return CSAQ_ERR_ARG;
  if (!aligned16(k_out) || !aligned16(v_out)) return CSAQ_ERR_UNSUPPORTED;
  if (n == 0) return CSAQ_OK;
  return by_layout(cache, D, LaunchRead{cache, B * Hkv, start, n, k_out, v_out, dtype, as_stream(stream)});
}

extern "C" int64_t csaq_kvq_attention_workspace_floats(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                                                       int64_t Lmax) {
  if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || Lmax <= 0) return -1;
  const Split split = split_of(B * Hkv, Lmax, 4);  // 8 bits take as much or none
  return split.partial ? B * Hkv * split.n * S * (Hq / Hkv) * (D + 2) : 0;
}

extern "C" int csaq_kvq_attention_launches(const csaq_kvq_cache* cache, int64_t B, int64_t Hkv, int64_t D) {
  const int rc = check_cache(cache, B, Hkv, D);
  if (rc) return rc;
  return split_of(B * Hkv, cache->Lmax, cache->bits).partial ? 2 : 1;
}

extern "C" int csaq_kvq_attention(const void* q, int64_t ldq, const csaq_kvq_cache* cache, const int32_t* pos0,
                                  int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, float scale, float* part,
                                  void* out, int64_t ldo, int dtype, void* stream) {
  const int rc = check_cache(cache, B, Hkv, D);
  if (rc) return rc;
  if (!q || !pos0 || !out || S <= 0 || Hq <= 0 || Hq % Hkv || ldq < Hq * D || ldo < Hq * D)
    return CSAQ_ERR_ARG;
  if (dtype != CSAQ_DT_F16 && dtype != CSAQ_DT_BF16) return CSAQ_ERR_ARG;
  const Split split = split_of(B * Hkv, cache->Lmax, cache->bits);
  if (!part && split.partial) return CSAQ_ERR_ARG;
  if (ldq % 8 || !aligned16(q) || ldo % 2 || reinterpret_cast<uintptr_t>(out) % 4 || reinterpret_cast<uintptr_t>(part) % 8 || S > 65535)
    return CSAQ_ERR_UNSUPPORTED;
  const AttnArgs a{q,
                   ldq,
                   cache->k_codes,
                   cache->v_codes,
                   cache->k_params,
                   cache->v_params,
                   pos0,
                   (int)S,
                   (int)Hq,
                   (int)Hkv,
                   (int)cache->Lmax,
                   split.chunk,
                   scale,
                   split.partial ? part : nullptr,
                   out,
                   ldo,
                   dtype == CSAQ_DT_BF16};
  return by_layout(cache, D, LaunchAttn{a, B, split, as_stream(stream)});
}
