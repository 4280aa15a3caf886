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

#include <atomic>

#include "common.cuh"

namespace csaq {
namespace {

constexpr int kMaxDev = 64;
constexpr uint32_t kZeroWord = 0x6400u;  // scale 0, zero point 0

__device__ __forceinline__ float word_scale(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// ── writing ─────────────────────────────────────────────────────────────────
// One quantisation group: s = bf16_up((max(x, 0) - min(x, 0)) / n), z = rint(-min / s),
// code = clamp(rint(x / s) + z, 0, n), every operation one fp32 rounding (no
// contraction), so that the codes are a definition and not a tolerance: values
// of 16-bit types meet the borders between codes exactly, and a correctly
// rounded quotient of them never crosses one. Zero is always representable. A
// group with a NaN or an infinity gets a NaN scale: all its values read back as
// NaN.
template <int BITS>
__device__ __forceinline__ uint32_t group_word(float lo, float hi, bool finite) {
  constexpr float n = (float)((1 << BITS) - 1);
  const float span = __fsub_rn(hi, lo);
  if (!finite) return 0x7fc00000u | kZeroWord;
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

// eight elements of each half of a head, codes of one half into 8 or 4 bytes
template <int BITS>
__device__ __forceinline__ void store_half(uint8_t* dst, const float* x, float s, float z) {
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = code_of<BITS>(x[i], s, z);
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

// D / 16 neighbouring threads take one head of one token: each holds elements
// i0..i0+7 and D/2+i0..D/2+i0+7, so that every rotation is its own and a
// group's minimum and maximum take log2(D / 16) shuffles.
template <typename T, int BITS, int D, int G>
__global__ void __launch_bounds__(256) kvq_write_kernel(const WriteArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int half = D / 2, TPH = D / 16;
  const int heads = (a.q ? a.Hq : 0) + 2 * a.Hkv;
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / TPH;
  const bool live = item < a.M * heads;
  const int64_t m = live ? item / heads : 0;
  int hh = live ? (int)(item - m * heads) : 0;
  const int i0 = (threadIdx.x % TPH) * 8;
  const int b = (int)(m / a.S);
  const int64_t pos = (int64_t)a.pos0[b] + (m - (int64_t)b * a.S);
  const bool is_q = a.q && hh < a.Hq;
  if (a.q && !is_q) hh -= a.Hq;
  const bool is_v = !is_q && hh >= a.Hkv;
  if (is_v) hh -= a.Hkv;
  const T* src = is_q ? reinterpret_cast<const T*>(a.q) + m * a.ldq
                      : (is_v ? reinterpret_cast<const T*>(a.v) + m * a.ldv : reinterpret_cast<const T*>(a.k) + m * a.ldk);
  src += (int64_t)hh * D;
  const bool turn = !is_v && a.cos_t != nullptr;
  // a position outside the cache or the tables: its keys and values are not
  // stored and its query is passed on unrotated
  const bool in_table = !a.cos_t || (pos >= 0 && pos < a.n_rope);
  const bool keep = live && pos >= 0 && pos < a.Lmax && in_table;
  float lo[8], hi[8];
  if (live) {
    const uint4 u = *reinterpret_cast<const uint4*>(src + i0);
    const uint4 w = *reinterpret_cast<const uint4*>(src + i0 + half);
    const T* ue = reinterpret_cast<const T*>(&u);
    const T* we = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = to_f32<T>(ue[i]), hi[i] = to_f32<T>(we[i]);
    if (turn && in_table) {
      float ca[8], sa[8], cb[8], sb[8];
      load8f(a.cos_t + pos * D + i0, ca);
      load8f(a.sin_t + pos * D + i0, sa);
      load8f(a.cos_t + pos * D + i0 + half, cb);
      load8f(a.sin_t + pos * D + i0 + half, sb);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x0 = lo[i], x1 = hi[i];
        lo[i] = __fsub_rn(__fmul_rn(x0, ca[i]), __fmul_rn(x1, sa[i]));
        hi[i] = __fadd_rn(__fmul_rn(x1, cb[i]), __fmul_rn(x0, sb[i]));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = hi[i] = 0.0f;
  }
  if (live && is_q) {
    uint4 u, w;
    T* ue = reinterpret_cast<T*>(&u);
    T* we = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) ue[i] = from_f32<T>(lo[i]), we[i] = from_f32<T>(hi[i]);
    T* dst = reinterpret_cast<T*>(a.q_out) + (m * a.Hq + hh) * D;
    *reinterpret_cast<uint4*>(dst + i0) = u;
    *reinterpret_cast<uint4*>(dst + i0 + half) = w;
  }
  // every thread takes part in the group shuffles (neighbours of a head are
  // always in one warp, and all of them are live or none)
  float mn0 = 0.0f, mx0 = 0.0f, mn1 = 0.0f, mx1 = 0.0f;
  bool ok0 = true, ok1 = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mn0 = fminf(mn0, lo[i]), mx0 = fmaxf(mx0, lo[i]), ok0 = ok0 && fabsf(lo[i]) <= 3.4e38f;
    mn1 = fminf(mn1, hi[i]), mx1 = fmaxf(mx1, hi[i]), ok1 = ok1 && fabsf(hi[i]) <= 3.4e38f;
  }
  if constexpr (G == D) {
    mn0 = mn1 = fminf(mn0, mn1);
    mx0 = mx1 = fmaxf(mx0, mx1);
    ok0 = ok1 = ok0 && ok1;
  }
  // a NaN or an infinity marks its group through an infinite maximum
  if (!ok0) mx0 = INFINITY;
  if (!ok1) mx1 = INFINITY;
#pragma unroll
  for (int o = 1; o < TPH; o <<= 1) {
    mn0 = fminf(mn0, __shfl_xor_sync(0xffffffffu, mn0, o));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
    if constexpr (G != D) {
      mn1 = fminf(mn1, __shfl_xor_sync(0xffffffffu, mn1, o));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
    }
  }
  if constexpr (G == D) mn1 = mn0, mx1 = mx0;
  if (!keep || is_q) return;
  constexpr int ROWB = D * BITS / 8, NG = D / G;
  const int64_t row = ((int64_t)b * a.Hkv + hh) * a.Lmax + pos;
  uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + row * ROWB;
  uint32_t* params = (is_v ? a.v_params : a.k_params) + row * NG;
  const uint32_t w0 = group_word<BITS>(mn0, mx0, mx0 <= 3.4e38f);
  const uint32_t w1 = G == D ? w0 : group_word<BITS>(mn1, mx1, mx1 <= 3.4e38f);
  // a group of zeros has scale 0 and may divide by anything
  const float s0 = word_scale(w0) != 0.0f ? word_scale(w0) : 1.0f, s1 = word_scale(w1) != 0.0f ? word_scale(w1) : 1.0f;
  store_half<BITS>(codes + i0 * BITS / 8, lo, s0, (float)((w0 & 0xffffu) - kZeroWord));
  store_half<BITS>(codes + (i0 + half) * BITS / 8, hi, s1, (float)((w1 & 0xffffu) - kZeroWord));
  if (i0 == 0) {
    params[0] = w0;
    if constexpr (G != D) params[1] = w1;
  }
}

// ── reading back ────────────────────────────────────────────────────────────
// A thread turns 16 codes into 16 values: one 16- or 8-byte load, two 16-byte
// stores (four for fp32). Positions [start, start + n) of every head; blockIdx.y
// strides over the (sequence, head) pairs and blockIdx.z picks keys or values.
template <typename T, int BITS, int D, int G>
__global__ void __launch_bounds__(256) kvq_read_kernel(const uint8_t* __restrict__ k_codes,
                                                       const uint32_t* __restrict__ k_params,
                                                       const uint8_t* __restrict__ v_codes,
                                                       const uint32_t* __restrict__ v_params, int64_t heads, int64_t Lmax,
                                                       int64_t start, int64_t n, T* __restrict__ k_out,
                                                       T* __restrict__ v_out) {
  pdl_wait();
  pdl_trigger();
  constexpr int ROWB = D * BITS / 8, NG = D / G, PER = D / 16;
  const bool is_v = blockIdx.z != 0 || !k_out;
  const uint8_t* codes = is_v ? v_codes : k_codes;
  const uint32_t* params = is_v ? v_params : k_params;
  T* out = is_v ? v_out : k_out;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * PER) return;
  const int64_t tok = i / PER;
  const int part = (int)(i - tok * PER);
  for (int64_t bh = blockIdx.y; bh < heads; bh += gridDim.y) {
    const int64_t row = bh * Lmax + start + tok;
    const uint32_t w = params[row * NG + part * 16 / G];
    const float s = word_scale(w), z = (float)((int)(w & 0xffffu) - (int)kZeroWord);
    float x[16];
    if constexpr (BITS == 8) {
      const uint4 c = *reinterpret_cast<const uint4*>(codes + row * ROWB + part * 16);
      const uint32_t cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = ((float)((cw[j / 4] >> (8 * (j % 4))) & 255u) - z) * s;
    } else {
      const uint2 c = *reinterpret_cast<const uint2*>(codes + row * ROWB + part * 8);
      const uint32_t cw[2] = {c.x, c.y};
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = ((float)((cw[j / 8] >> (4 * (j % 8))) & 15u) - z) * s;
    }
    T* dst = out + (bh * n + tok) * D + part * 16;
    constexpr int VE = 16 / (int)sizeof(T);  // elements of a 16-byte store
#pragma unroll
    for (int v = 0; v < 16 / VE; ++v) {
      uint4 u;
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int j = 0; j < VE; ++j) e[j] = from_f32<T>(x[v * VE + j]);
      reinterpret_cast<uint4*>(dst)[v] = u;
    }
  }
}

// ── attention ───────────────────────────────────────────────────────────────
// Token (b, s) attends keys 0 .. pos0[b] + s. With codes c, zero points z and
// scales s, a score is s_k (q . (c_k - z_k)) and an output sum_j (p_j s_j)(c_j - z_j):
// the scales leave the products, which run on the tensor cores over exact small
// integers in fp16 with fp32 sums (mma.sync m16n8k16: at most 32 query rows share
// a key, far below the rate at which the codes arrive, and the operands come from
// registers without a second trip through shared memory). Keys take the M side of
// S^T = K q^T and head elements the M side of O^T = V^T P^T, so that 8 query rows
// fill an instruction. q enters as fp16 after a power of two per row brings its
// largest magnitude to [2^14, 2^15): exact for fp16 and bf16 q, except that
// elements below 2^-31 of the row's largest lose bits, under 2^-39 of it.
//
// A CTA takes one chunk of `chunk` keys of one KV head for up to 8 NT query rows;
// each of its 8 warps takes every eighth tile of 16 keys through a ring of its own
// (16-byte asynchronous copies; no barrier in the loop) and keeps its own softmax
// state. The states are joined in warp order, then the chunks' in chunk order by
// the last CTA of a head (a ticket; no waiting). Chunk, tile and joining order
// depend on key indices and the launch's fixed sizes (B Hkv, Lmax) alone: a
// token's result does not depend on how many tokens share its step.
constexpr int kWarps = 8;
constexpr int kTile = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHead = 7.0f, kTop = 15.0f;  // exponents of the weights (see the state's comment)

struct AttnArgs {
  const void* q;
  int64_t ldq;
  const uint8_t *k_codes, *v_codes;
  const uint32_t *k_params, *v_params;
  const int32_t* pos0;
  int S, Hq, Hkv, Lmax, chunk;
  float scale;
  float* part;
  int32_t* tickets;
  void* out;
  int64_t ldo;
  int bf16;
};

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
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
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
// 64 + z from 1024 + z (both halves), for nibbles read four bits up in the mantissa
__device__ __forceinline__ uint32_t zero_high(uint32_t z) { return ((z & 0x000f000fu) << 4) | 0x54005400u; }

template <int BITS, int D, int G, int NT>
struct Attn {
  static constexpr int ROWB = D * BITS / 8;       // code bytes of a key
  static constexpr int NG = D / G, NB = D / 64;   // parameter groups, 64-element blocks
  static constexpr int BPG = G / 64;              // blocks of a group
  static constexpr int KV = kTile * ROWB;         // code bytes of a tile's keys (or values)
  static constexpr int PW = kTile * NG;           // parameter words of a tile's keys (or values)
  static constexpr int STAGE = 2 * KV + 8 * PW;
  static constexpr bool QSMEM = NT > 1;           // query operands reread from shared memory
  static constexpr int CTAS = NT <= 2 ? 2 : 1;    // per SM: accumulators take 16 D / 64 NT registers a thread
  // ring depth: about 100 KB a CTA at two per SM, 200 KB at one, 8 stages at most
  static constexpr int FIT = (CTAS == 2 ? 104 : 200) * 1024 / (kWarps * STAGE);
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  static constexpr int RING = kWarps * STAGES * STAGE;
  static constexpr int JOIN = kWarps * 8 * NT * (D + 2) * 4;
  static constexpr int QBYTES = 8 * NT * D * 2;   // fp16 query rows, then their fragments in place of the rows
  static constexpr int SMEM = (RING > JOIN ? RING : JOIN) + QBYTES;
  static constexpr int swz_k(int key) { return ROWB == 128 ? (key & 1) << 2 : (ROWB == 64 ? key & 2 : 0); }
  static constexpr int swz_v(int key) { return ROWB == 128 ? key & 6 : (ROWB == 64 ? (key & 6) >> 1 : 0); }
};

template <typename C>
__device__ __forceinline__ void issue_tile(uint32_t dst, const uint8_t* kc, const uint8_t* vc, const uint32_t* kp,
                                           const uint32_t* vp, int n_keys, int lane) {
  constexpr int CPR = C::ROWB / 16;  // 16-byte pieces of a row
#pragma unroll
  for (int e = lane; e < kTile * CPR; e += 32) {
    const int key = e / CPR, c = e % CPR;
    if (key < n_keys) {
      cp16(dst + key * C::ROWB + ((c ^ C::swz_k(key)) * 16), kc + e * 16);
      cp16(dst + C::KV + key * C::ROWB + ((c ^ C::swz_v(key)) * 16), vc + e * 16);
    }
  }
  // parameters: PW / 4 pieces each; a piece holds 4 / NG keys and lies inside the
  // buffer when its first key does (Lmax is a multiple of 16)
  constexpr int PP = C::PW / 4;
  if (lane < 2 * PP) {
    const bool is_v = lane >= PP;
    const int c = is_v ? lane - PP : lane;
    if (c * 4 / C::NG < n_keys) cp16(dst + 2 * C::KV + is_v * C::PW * 4 + c * 16, (is_v ? vp : kp) + c * 4);
  }
}

// fp16 operand registers of eight (4-bit) or four (8-bit) codes in `w`, minus the
// zero point: for 8 bits {(0,1), (2,3)}, for 4 bits {(0,4), (1,5), (2,6), (3,7)}
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

template <int BITS, int D, int G, int NT>
__global__ void __launch_bounds__(kWarps * 32, Attn<BITS, D, G, NT>::CTAS) kvq_attention_kernel(const AttnArgs a) {
  using C = Attn<BITS, D, G, NT>;
  constexpr int NB = C::NB, NG = C::NG;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float row_mul[8 * NT];
  __shared__ int is_last;
  const int bh = blockIdx.x, sp = blockIdx.y, n_split = gridDim.y;
  const int b = bh / a.Hkv, h = bh % a.Hkv;
  const int Gq = a.Hq / a.Hkv, R = a.S * Gq;  // query heads per KV head, query rows of the head
  const int r0 = blockIdx.z * 8 * NT, rows = min(8 * NT, R - r0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_trigger();
  const int64_t p0 = a.pos0[b];
  const int64_t end = p0 + a.S;
  const int len = (int)(end < 0 ? 0 : (end > a.Lmax ? a.Lmax : end));  // keys visible to the last token
  const int n_act = len > a.chunk ? (len + a.chunk - 1) / a.chunk : 1;
  if (sp >= n_act) return;
  const int k0 = sp * a.chunk, k1 = min(len, k0 + a.chunk);

  // this warp's copies go out before the queries are prepared
  const int64_t head_row = (int64_t)bh * a.Lmax;
  uint8_t* ring = smem + warp * (C::STAGES * C::STAGE);
  const uint32_t ring_a = smem_addr(ring);
  const int first = k0 + warp * kTile;
  const int n_tiles = first < k1 ? (k1 - first + kWarps * kTile - 1) / (kWarps * kTile) : 0;
  auto issue = [&](int i) {
    if (i < n_tiles) {
      const int key = first + i * kWarps * kTile;
      const int64_t row = head_row + key;
      issue_tile<C>(ring_a + (i % C::STAGES) * C::STAGE, a.k_codes + row * C::ROWB, a.v_codes + row * C::ROWB,
                    a.k_params + row * NG, a.v_params + row * NG, k1 - key, lane);
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) issue(i);

  // query rows: one warp a row, scaled by a power of two into fp16
  uint8_t* qbase = smem + C::SMEM - C::QBYTES;
  __half* qs = reinterpret_cast<__half*>(qbase);
  for (int r = warp; r < 8 * NT; r += kWarps) {
    float x[D / 32], big = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) x[i] = 0.0f;
    if (r < rows) {
      const int rr = r0 + r, s = rr / Gq, hq = h * Gq + rr % Gq;
      const int64_t at = ((int64_t)b * a.S + s) * a.ldq + (int64_t)hq * D + lane * (D / 32);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        x[i] = a.bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.q)[at + i])
                      : __half2float(reinterpret_cast<const __half*>(a.q)[at + i]);
        big = fmaxf(big, fabsf(x[i]));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
    const int e = (int)(__float_as_uint(big) >> 23) - 127;  // floor(log2), -127 for zero and subnormals
    const int up = min(14 - e, 126);
    const float f = __uint_as_float((uint32_t)(up + 127) << 23);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) qs[r * D + lane * (D / 32) + i] = __float2half_rn(x[i] * f);
    if (lane == 0) row_mul[r] = a.scale * kLog2e * __uint_as_float((uint32_t)(127 - up) << 23);
  }
  __syncthreads();
  // B operands of the score product: step i of block nb holds the elements that
  // the K operand below has there, for query row g of n-tile nt
  auto q_frag = [&](int nt, int st, uint32_t& f0, uint32_t& f1) {
    const __half* q = qs + (nt * 8 + g) * D + (st / 4) * 64 + t * 16;
    const int i = st % 4;
    if constexpr (BITS == 8) {
      f0 = *reinterpret_cast<const uint32_t*>(q + 4 * i);
      f1 = *reinterpret_cast<const uint32_t*>(q + 4 * i + 2);
    } else {
      const __half* e = q + 8 * (i / 2) + 2 * (i % 2);
      const uint32_t lo = *reinterpret_cast<const uint32_t*>(e), up = *reinterpret_cast<const uint32_t*>(e + 4);
      f0 = prmt(lo, up, 0x5410);
      f1 = prmt(lo, up, 0x7632);
    }
  };
  uint32_t qf[C::QSMEM ? 1 : NB * 4][2];
  if constexpr (C::QSMEM) {
    // the fragments replace the rows, [step][n-tile][lane]: a warp turns one step
    const int st = warp % (NB * 4);
    uint32_t f[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) q_frag(nt, st, f[nt][0], f[nt][1]);
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      reinterpret_cast<uint2*>(qbase)[(st * NT + nt) * 32 + lane] = make_uint2(f[nt][0], f[nt][1]);
    __syncthreads();
  } else {
#pragma unroll
    for (int st = 0; st < NB * 4; ++st) q_frag(0, st, qf[st][0], qf[st][1]);
  }
  float mul[NT][2];  // softmax scale, log2 e and the power of two of rows 2t, 2t + 1
  int lim[NT][2];    // keys visible to them
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = nt * 8 + 2 * t + j;
      mul[nt][j] = row_mul[r];
      const int64_t l = p0 + min(r0 + r, R - 1) / Gq + 1;
      lim[nt][j] = (int)(l < 0 ? 0 : (l > len ? len : l));
    }
  const int64_t l0 = p0 + r0 / Gq + 1;
  const int lim_first = (int)(l0 < 0 ? 0 : (l0 > len ? len : l0));  // every row of the block sees the keys below

  // The state of a row: a reference m, l = sum_j 2^(s_j - m), o = sum_j 2^(s_j - m) s_vj (c_j - z_j).
  // The weights 2^(s_j - m) s_vj are rounded to fp16 for the product: 2^-11 relative
  // each, below the output's own rounding for bf16 and the size of it for fp16. So
  // that they use fp16's range whatever the scale of V, m follows the largest
  // s_j + log2 s_vj: that weight is 2^kHead, and m moves only when a tile exceeds
  // 2^kTop <= 65504. Weights keep their full precision down to 2^-21 of the largest
  // and vanish below 2^-32 of it, which a million of them do not make up.
  float m[NT][2], l[NT][2], o[NT][NB * 4][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < NB * 4; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
  }

  for (int it = 0; it < n_tiles; ++it) {
    cp_wait<C::STAGES - 2>();
    __syncwarp();  // the tile is in shared memory for every lane, and the previous one has been read
    issue(it + C::STAGES - 1);
    const uint8_t* stage = ring + (it % C::STAGES) * C::STAGE;
    const int key0 = first + it * kWarps * kTile;
    const uint32_t* kpw = reinterpret_cast<const uint32_t*>(stage + 2 * C::KV);
    const uint32_t* vpw = kpw + C::PW;
    const bool whole = key0 + kTile <= lim_first;  // no key of the tile is masked for any row

    // scores: keys g and g + 8 of the tile, rows 2t and 2t + 1
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      const uint32_t wa = kpw[g * NG + grp], wb = kpw[(g + 8) * NG + grp];
      const uint32_t za = prmt(wa, wa, 0x1010), zb = prmt(wb, wb, 0x1010);
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
#pragma unroll
      for (int bb = 0; bb < C::BPG; ++bb) {
        const int nb = grp * C::BPG + bb;
        uint32_t A[4][4];
        if constexpr (BITS == 8) {
          const uint4 ca = *reinterpret_cast<const uint4*>(stage + g * C::ROWB + (((nb * 4 + t) ^ C::swz_k(g)) * 16));
          const uint4 cb =
              *reinterpret_cast<const uint4*>(stage + (g + 8) * C::ROWB + (((nb * 4 + t) ^ C::swz_k(g + 8)) * 16));
          const uint32_t xa[4] = {ca.x, ca.y, ca.z, ca.w}, xb[4] = {cb.x, cb.y, cb.z, cb.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t ra[2], rb[2];
            codes8(xa[i], za, ra);
            codes8(xb[i], zb, rb);
            A[i][0] = ra[0], A[i][1] = rb[0], A[i][2] = ra[1], A[i][3] = rb[1];
          }
        } else {
          const uint32_t zah = zero_high(za), zbh = zero_high(zb);
          const int c = nb * 2 + t / 2, in = (t % 2) * 8;
          const uint2 ca = *reinterpret_cast<const uint2*>(stage + g * C::ROWB + ((c ^ C::swz_k(g)) * 16) + in);
          const uint2 cb =
              *reinterpret_cast<const uint2*>(stage + (g + 8) * C::ROWB + ((c ^ C::swz_k(g + 8)) * 16) + in);
          const uint32_t xa[2] = {ca.x, ca.y}, xb[2] = {cb.x, cb.y};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t ra[4], rb[4];
            codes4(xa[i], za, zah, ra);
            codes4(xb[i], zb, zbh, rb);
            A[2 * i][0] = ra[0], A[2 * i][1] = rb[0], A[2 * i][2] = ra[1], A[2 * i][3] = rb[1];
            A[2 * i + 1][0] = ra[2], A[2 * i + 1][1] = rb[2], A[2 * i + 1][2] = ra[3], A[2 * i + 1][3] = rb[3];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if constexpr (C::QSMEM) {
              const uint2 f = reinterpret_cast<const uint2*>(qbase)[((nb * 4 + i) * NT + nt) * 32 + lane];
              const uint32_t B[2] = {f.x, f.y};
              mma16816(acc[nt], A[i], B);
            } else {
              mma16816(acc[nt], A[i], qf[nb * 4 + i]);
            }
          }
      }
      const float sa = word_scale(wa), sb = word_scale(wb);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sc[nt][0] = fmaf(acc[nt][0], sa, sc[nt][0]);
        sc[nt][1] = fmaf(acc[nt][1], sa, sc[nt][1]);
        sc[nt][2] = fmaf(acc[nt][2], sb, sc[nt][2]);
        sc[nt][3] = fmaf(acc[nt][3], sb, sc[nt][3]);
      }
    }
    // V's scales of keys g and g + 8; a key behind the last one has no parameters
    float va[NG], vb[NG], ea = 0.0f, eb = 0.0f;
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      va[grp] = word_scale(vpw[g * NG + grp]);
      vb[grp] = word_scale(vpw[(g + 8) * NG + grp]);
      ea = fmaxf(ea, va[grp]);
      eb = fmaxf(eb, vb[grp]);
    }
    ea = fmaxf(lg2(ea), -80.0f);  // 2^(s - m) stays below 2^95, a sum of them finite
    eb = fmaxf(lg2(eb), -80.0f);
    bool over = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sc[nt][j] *= mul[nt][j];
        sc[nt][2 + j] *= mul[nt][j];
        if (!whole) {
          if (key0 + g >= lim[nt][j]) sc[nt][j] = -INFINITY;
          if (key0 + g + 8 >= lim[nt][j]) sc[nt][2 + j] = -INFINITY;
        }
        over = over || fmaxf(sc[nt][j] + ea, sc[nt][2 + j] + eb) > m[nt][j] + kTop;
      }
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = fmaxf(sc[nt][j] + ea, sc[nt][2 + j] + eb);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          if (top > m[nt][j] + kTop) {  // a row moves by its own scores alone
            const float to = top - kHead;
            const float f = ex2(m[nt][j] - to);  // 0 from -inf
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
    // weights, and their B operands (a transposition of 8 keys x 8 rows)
    uint32_t P[NG][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float p[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float ref = m[nt][j] == -INFINITY ? 0.0f : m[nt][j];  // nothing seen yet: every weight is 0
        p[j] = ex2(sc[nt][j] - ref);
        p[2 + j] = ex2(sc[nt][2 + j] - ref);
        l[nt][j] += p[j] + p[2 + j];
      }
#pragma unroll
      for (int grp = 0; grp < NG; ++grp) {
        float wa0 = p[0] * va[grp], wa1 = p[1] * va[grp], wb0 = p[2] * vb[grp], wb1 = p[3] * vb[grp];
        if (!whole) {  // a masked key's scale may be anything
          wa0 = sc[nt][0] == -INFINITY ? 0.0f : wa0;
          wa1 = sc[nt][1] == -INFINITY ? 0.0f : wa1;
          wb0 = sc[nt][2] == -INFINITY ? 0.0f : wb0;
          wb1 = sc[nt][3] == -INFINITY ? 0.0f : wb1;
        }
        P[grp][nt][0] = transpose8x8(pack2(wa0, wa1));
        P[grp][nt][1] = transpose8x8(pack2(wb0, wb1));
      }
    }
    // outputs: V's codes of keys 2t, 2t + 1, 2t + 8, 2t + 9, head elements 8g.. of each block
#pragma unroll
    for (int grp = 0; grp < NG; ++grp) {
      uint32_t w0 = vpw[(2 * t) * NG + grp], w1 = vpw[(2 * t + 1) * NG + grp];
      uint32_t w2 = vpw[(2 * t + 8) * NG + grp], w3 = vpw[(2 * t + 9) * NG + grp];
      if (!whole) {  // the zero points behind the last key must be numbers
        w0 = key0 + 2 * t < k1 ? w0 : kZeroWord;
        w1 = key0 + 2 * t + 1 < k1 ? w1 : kZeroWord;
        w2 = key0 + 2 * t + 8 < k1 ? w2 : kZeroWord;
        w3 = key0 + 2 * t + 9 < k1 ? w3 : kZeroWord;
      }
      const uint32_t z01 = prmt(w0, w1, 0x5410), z23 = prmt(w2, w3, 0x5410);
#pragma unroll
      for (int bb = 0; bb < C::BPG; ++bb) {
        const int nb = grp * C::BPG + bb;
        uint32_t E[8][2];  // element e: keys (2t, 2t + 1), (2t + 8, 2t + 9)
        const uint8_t* vs = stage + C::KV;
        if constexpr (BITS == 8) {
          const int c = nb * 4 + g / 2, in = (g % 2) * 8;
          auto at = [&](int key) {
            return *reinterpret_cast<const uint2*>(vs + key * C::ROWB + ((c ^ C::swz_v(key)) * 16) + in);
          };
          const uint2 x0 = at(2 * t), x1 = at(2 * t + 1), x2 = at(2 * t + 8), x3 = at(2 * t + 9);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t y0 = w ? x0.y : x0.x, y1 = w ? x1.y : x1.x, y2 = w ? x2.y : x2.x, y3 = w ? x3.y : x3.x;
            uint32_t r[2];
            codes8(prmt(y0, y1, 0x5140), z01, r);
            E[4 * w][0] = r[0], E[4 * w + 1][0] = r[1];
            codes8(prmt(y0, y1, 0x7362), z01, r);
            E[4 * w + 2][0] = r[0], E[4 * w + 3][0] = r[1];
            codes8(prmt(y2, y3, 0x5140), z23, r);
            E[4 * w][1] = r[0], E[4 * w + 1][1] = r[1];
            codes8(prmt(y2, y3, 0x7362), z23, r);
            E[4 * w + 2][1] = r[0], E[4 * w + 3][1] = r[1];
          }
        } else {
          const int c = nb * 2 + g / 4, in = (g % 4) * 4;
          auto at = [&](int key) {
            return *reinterpret_cast<const uint32_t*>(vs + key * C::ROWB + ((c ^ C::swz_v(key)) * 16) + in);
          };
          const uint32_t x0 = at(2 * t), x1 = at(2 * t + 1), x2 = at(2 * t + 8), x3 = at(2 * t + 9);
          const uint32_t z01h = zero_high(z01), z23h = zero_high(z23);
          uint32_t r[4];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t sel = w ? 0x7632 : 0x5410;
            codes4(prmt(x0, x1, sel), z01, z01h, r);
#pragma unroll
            for (int e = 0; e < 4; ++e) E[4 * w + e][0] = r[e];
            codes4(prmt(x2, x3, sel), z23, z23h, r);
#pragma unroll
            for (int e = 0; e < 4; ++e) E[4 * w + e][1] = r[e];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t A[4] = {E[2 * i][0], E[2 * i + 1][0], E[2 * i][1], E[2 * i + 1][1]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][nb * 4 + i], A, P[grp][nt]);
        }
      }
    }
  }
  cp_wait<0>();
  __syncthreads();  // every warp has read its last tile: the ring becomes the joining buffer

  // states of the warps: [warp][row][D + 2] = o, m, l
  float* join = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
      l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
      l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
      float* to = join + (warp * 8 * NT + nt * 8 + 2 * t + j) * (D + 2);
#pragma unroll
      for (int i = 0; i < NB * 4; ++i)
        *reinterpret_cast<float2*>(to + (i / 4) * 64 + g * 8 + (i % 4) * 2) = make_float2(o[nt][i][j], o[nt][i][2 + j]);
      if (g == 0) to[D] = m[nt][j], to[D + 1] = l[nt][j];
    }
  }
  __syncthreads();
  auto store = [&](int r, int d, float2 v) {  // two neighbouring head elements of row r0 + r
    const int rr = r0 + r, s = rr / Gq, hq = h * Gq + rr % Gq;
    const int64_t at = ((int64_t)b * a.S + s) * a.ldo + (int64_t)hq * D + d;
    if (a.bf16)
      *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<__nv_bfloat16*>(a.out) + at) = __floats2bfloat162_rn(v.x, v.y);
    else
      *reinterpret_cast<__half2*>(reinterpret_cast<__half*>(a.out) + at) = __floats2half2_rn(v.x, v.y);
  };
  // [bh][split][row][D + 2]
  float* part = a.part + ((int64_t)bh * n_split * R + r0) * (D + 2);
  for (int e = threadIdx.x; e < rows * (D / 2); e += kWarps * 32) {
    const int r = e / (D / 2), d = (e % (D / 2)) * 2;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, join[(w * 8 * NT + r) * (D + 2) + D]);
    float L = 0.0f;
    float2 acc = make_float2(0.0f, 0.0f);
    if (top != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* from = join + (w * 8 * NT + r) * (D + 2);
        const float f = ex2(from[D] - top);
        const float2 v = *reinterpret_cast<const float2*>(from + d);
        L = fmaf(from[D + 1], f, L);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
      }
    } else {  // no key, or scores that are all NaN
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* from = join + (w * 8 * NT + r) * (D + 2);
        const float2 v = *reinterpret_cast<const float2*>(from + d);
        L += from[D + 1], acc.x += v.x, acc.y += v.y;
      }
    }
    if (n_act == 1) {
      const float inv = L != 0.0f ? 1.0f / L : 0.0f;  // a row that sees no key is 0
      store(r, d, make_float2(acc.x * inv, acc.y * inv));
    } else {
      float* to = part + ((int64_t)sp * R + r) * (D + 2);
      *reinterpret_cast<float2*>(to + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(to + D) = make_float2(top, L);
    }
  }
  if (n_act == 1) return;
  __threadfence();
  __syncthreads();
  int32_t* ticket = a.tickets + (int64_t)bh * gridDim.z + blockIdx.z;
  if (threadIdx.x == 0) is_last = atomicAdd(ticket, 1) == n_act - 1;
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  for (int e = threadIdx.x; e < rows * (D / 2); e += kWarps * 32) {
    const int r = e / (D / 2), d = (e % (D / 2)) * 2;
    const float* from = part + (int64_t)r * (D + 2);
    const int64_t step = (int64_t)R * (D + 2);
    float top = -INFINITY;
    for (int p = 0; p < n_act; ++p) top = fmaxf(top, __ldcg(from + p * step + D));
    const float ref = top == -INFINITY ? 0.0f : top;
    float L = 0.0f;
    float2 acc = make_float2(0.0f, 0.0f);
    for (int p = 0; p < n_act; ++p) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(from + p * step + D));
      const float2 v = __ldcg(reinterpret_cast<const float2*>(from + p * step + d));
      const float f = top == -INFINITY ? 1.0f : ex2(ml.x - ref);
      L = fmaf(ml.y, f, L);
      acc.x = fmaf(v.x, f, acc.x);
      acc.y = fmaf(v.y, f, acc.y);
    }
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    store(r, d, make_float2(acc.x * inv, acc.y * inv));
  }
  if (threadIdx.x == 0) *ticket = 0;
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
    const int64_t blocks = (a.M * heads * (D / 16) + 255) / 256;
    if (blocks > INT32_MAX) return CSAQ_ERR_UNSUPPORTED;
    if (dtype == CSAQ_DT_BF16)
      return launch_pdl(kvq_write_kernel<__nv_bfloat16, BITS, D, G>, dim3((unsigned)blocks), dim3(256), 0, st, a);
    return launch_pdl(kvq_write_kernel<__half, BITS, D, G>, dim3((unsigned)blocks), dim3(256), 0, st, a);
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
    const int64_t bx = (n * (D / 16) + 255) / 256;
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

// Keys per CTA, from B * Hkv and Lmax alone (so that a step's token count does
// not move the chunk borders): the smallest power of two from 128 (one tile a
// warp) that cuts a full cache into at most kMaxItems pieces.
constexpr int64_t kMaxItems = 4 * 2 * 148;
int chunk_keys(int64_t heads, int64_t Lmax) {
  int64_t c = kWarps * kTile;
  while (heads * ((Lmax + c - 1) / c) > kMaxItems && c < Lmax) c *= 2;
  return (int)c;
}
int64_t n_splits(int64_t heads, int64_t Lmax) {
  const int64_t c = chunk_keys(heads, Lmax);
  return (Lmax + c - 1) / c;
}

struct LaunchAttn {
  const AttnArgs& a;
  int64_t heads;
  cudaStream_t st;
  template <int BITS, int D, int G, int NT>
  int go() const {
    using C = Attn<BITS, D, G, NT>;
    static_assert(C::STAGES >= 3, "the ring needs three stages");
    static std::atomic<uint64_t> ready{0};  // devices on which the kernel's shared memory is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) {
      set_last_cuda_error(e);
      return CSAQ_ERR_CUDA;
    }
    if (dev < 0 || dev >= kMaxDev) return CSAQ_ERR_UNSUPPORTED;
    auto kern = kvq_attention_kernel<BITS, D, G, NT>;
    if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
      if (e != cudaSuccess) {
        set_last_cuda_error(e);
        (void)cudaGetLastError();
        return CSAQ_ERR_CUDA;
      }
      ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    const int64_t R = (int64_t)a.S * (a.Hq / a.Hkv);
    const dim3 grid((unsigned)heads, (unsigned)n_splits(heads, a.Lmax), (unsigned)((R + 8 * NT - 1) / (8 * NT)));
    return launch_pdl(kern, grid, dim3(kWarps * 32), C::SMEM, st, a);
  }
  template <int BITS, int D, int G>
  int run() const {
    const int64_t R = (int64_t)a.S * (a.Hq / a.Hkv);
    if (R <= 8) return go<BITS, D, G, 1>();
    if (R <= 16) return go<BITS, D, G, 2>();
    if (R <= 24) return go<BITS, D, G, 3>();
    return go<BITS, D, G, 4>();
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
  return B * Hkv * n_splits(B * Hkv, Lmax) * S * (Hq / Hkv) * (D + 2);
}

extern "C" int64_t csaq_kvq_attention_tickets(int64_t B, int64_t S, int64_t Hq, int64_t Hkv) {
  if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return -1;
  return B * Hkv * ((S * (Hq / Hkv) + 7) / 8);
}

extern "C" int csaq_kvq_attention(const void* q, int64_t ldq, const csaq_kvq_cache* cache, const int32_t* pos0,
                                  int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, float scale, float* part,
                                  int32_t* tickets, void* out, int64_t ldo, int dtype, void* stream) {
  const int rc = check_cache(cache, B, Hkv, D);
  if (rc) return rc;
  if (!q || !pos0 || !part || !tickets || !out || S <= 0 || Hq <= 0 || Hq % Hkv || ldq < Hq * D || ldo < Hq * D)
    return CSAQ_ERR_ARG;
  if (dtype != CSAQ_DT_F16 && dtype != CSAQ_DT_BF16) return CSAQ_ERR_ARG;
  const int64_t heads = B * Hkv;
  if (ldo % 2 || reinterpret_cast<uintptr_t>(out) % 4 || reinterpret_cast<uintptr_t>(part) % 8 || S > 65535 ||
      S * (Hq / Hkv) > 65535 * 32 || n_splits(heads, cache->Lmax) > 65535)
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
                   chunk_keys(heads, cache->Lmax),
                   scale,
                   part,
                   tickets,
                   out,
                   ldo,
                   dtype == CSAQ_DT_BF16};
  return by_layout(cache, D, LaunchAttn{a, heads, as_stream(stream)});
}
