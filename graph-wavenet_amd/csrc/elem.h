// Shared by the position-wise layers (linear.hip, layernorm.hip, dropout.hip): the element types,
// vector access at any element alignment, the activations and the dropout generator.
#pragma once
#include "gwn_internal.h"

namespace elem {

typedef _Float16 f16;
typedef __bf16 bf16;

// 16 bytes of elements: one global_load_dwordx4 per lane
template <typename T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };

// n-element access aligned to the element only (rows of odd widths start anywhere): the packed
// struct tells the compiler the alignment, and gfx950 loads and stores dwords at any byte address
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load(const T* p) {
  return *reinterpret_cast<const Pack<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const Pack<T, N>& v) {
  *reinterpret_cast<Pack<T, N>*>(p) = v;
}

// The same where a load's latency counts and rows are of odd lengths: a 16-byte load off a 4-byte border
// takes more than twice as long, so 16-bit values are loaded by the whole dwords that hold them and
// shifted into place (12 rows of 1999 by 1030 columns in f16: 13.4 -> 8.5 us; where many rows stream, as in
// layer norm, the plain load is the faster one).
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_odd(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return load<T, N>(p);
  } else {
    const unsigned long long a = (unsigned long long)p;
    const unsigned sh = (unsigned)(a & 2) * 8;
    const unsigned* d = (const unsigned*)(a & ~3ull);
    const Pack<unsigned, N / 2> lo = load<unsigned, N / 2>(d);
    const unsigned last = d[N / 2 - (sh ? 0 : 1)];  // never a dword without a value
    Pack<T, N> r;
    unsigned o[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) o[i] = __builtin_amdgcn_alignbit(i + 1 < N / 2 ? lo.v[i + 1] : last, lo.v[i], sh);
    __builtin_memcpy(&r, o, sizeof(r));
    return r;
  }
}

// ---- dropout ---------------------------------------------------------------------------------
// Counter based: element i of a tensor is kept by the mask of (seed, salt) iff u24(i) >= thr, thr =
// ceil(p 2^24).  The 64-bit key is two rounds of the SplitMix64 finaliser (Steele, Lea and Flood
// 2014) over seed, salt and the high half of i; its low word starts the 32-bit mix of the low half
// (the constants of gwn_mix32), its high word enters between that mix's two multiplies, so that two
// keys' streams are not shifts of one another.  Three multiplies per element, no memory: the mask is
// the same in every kernel that applies or differentiates it.
struct Drop {
  const unsigned long long* seed_ptr;
  unsigned long long salt;
  unsigned thr;  // 0: no dropout
  float scale;   // 1 / (1 - p); 0 for p = 1
};

__host__ __device__ inline unsigned long long mix64(unsigned long long v) {
  v = (v ^ (v >> 30)) * 0xBF58476D1CE4E5B9ull;
  v = (v ^ (v >> 27)) * 0x94D049BB133111EBull;
  return v ^ (v >> 31);
}

struct DropKey {
  unsigned long long base;
  unsigned hi, k0, k1;
  __device__ __forceinline__ void rekey(unsigned h) {
    const unsigned long long k = mix64(base + h);
    hi = h;
    k0 = (unsigned)k;
    k1 = (unsigned)(k >> 32);
  }
  __device__ __forceinline__ void init(const Drop& d, unsigned long long i) {
    base = mix64(*d.seed_ptr + 0x9E3779B97F4A7C15ull * (d.salt + 1));
    // a wave's elements share the high half but where it steps: keyed once, on the scalar unit
    rekey(__builtin_amdgcn_readfirstlane((unsigned)(i >> 32)));
  }
  __device__ __forceinline__ void seek(unsigned long long i) {
    if ((unsigned)(i >> 32) != hi) rekey((unsigned)(i >> 32));
  }
  // of element i, the high half of which seek() has set
  __device__ __forceinline__ bool keep(unsigned lo, unsigned thr) const {
    unsigned h = lo * 0x9E3779B1u + k0;
    h ^= h >> 16;
    h *= 0x7FEB352Du;
    h ^= h >> 15;
    h += k1;
    h *= 0x846CA68Bu;
    h ^= h >> 16;
    return (h >> 8) >= thr;
  }
};

// ---- activations -----------------------------------------------------------------------------
// FAST (16-bit results): exp and reciprocal by the hardware's instructions, gelu's Phi by normal_tail.  Products that can meet
// an infinity and a zero take the multiply that gives zero there, so that every activation and slope
// has its limits at both ends, without a branch; a NaN stays one.
template <bool FAST> __device__ __forceinline__ float exp_(float x) {
  return FAST ? __builtin_amdgcn_exp2f(1.44269504f * x) : expf(x);
}
template <bool FAST> __device__ __forceinline__ float rcp_(float x) {
  return FAST ? __builtin_amdgcn_rcpf(x) : 1.0f / x;
}
// The instruction v_mul_legacy_f32, by the compiler's intrinsic (it has no builtin): the compiler places
// the wait that a use of an exp or rcp result needs.
extern "C" __device__ float gwn_fmul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ float mul0(float a, float b) { return gwn_fmul_legacy(a, b); }

// The normal distribution's tail Phi(-a), a >= 0, over e = exp(-a^2 / 2): a polynomial in t = 1 / (1 + 0.3025 a)
// without a constant term, fitted to erfcx(a / sqrt 2) / 2 on 0 .. 14 by Lawson's iteration (weighted least squares whose
// weights grow with the error).  Its relative error in fp32 is at most 1.6e-6 up to a = 1 and 1.3e-5 beyond, a fortieth of half
// a step of f16, so that gelu keeps bf16's precision down the negative tail too, where a formula of
// bounded absolute error does not (Abramowitz and Stegun 7.1.26, one term shorter: 1.5% off at z = -9).
__device__ __forceinline__ float normal_tail(float a) {
  const float t = rcp_<true>(1.0f + 0.3025f * a);
  return t * (0.121032165f +
              t * (0.11519542f + t * (0.142840961f + t * (-0.0121391147f + t * (0.211066591f - t * 0.0779966099f)))));
}

// the normal distribution's Phi(z); e = exp(-z^2 / 2)
template <bool FAST> __device__ __forceinline__ float normal_cdf(float z, float e) {
  if (!FAST) return 0.5f * erfcf(-0.70710678f * z);
  const float tail = normal_tail(fabsf(z)) * e;
  return z < 0.0f ? tail : 1.0f - tail;
}
// 2 sqrt(2/pi) (z + 0.044715 z^3): gelu_tanh is z / (1 + exp(-u))
__device__ __forceinline__ float gelu_u(float z) { return z * (1.5957691216f + 0.0713548163f * z * z); }

template <bool FAST, int ACT> __device__ __forceinline__ float act_value(float z) {
  if (ACT == GWN_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
  if (ACT == GWN_ACT_GELU) return mul0(z, normal_cdf<FAST>(z, FAST ? exp_<FAST>(-0.5f * z * z) : 0.0f));
  if (ACT == GWN_ACT_GELU_TANH) return mul0(z, rcp_<FAST>(1.0f + exp_<FAST>(-gelu_u(z))));
  if (ACT == GWN_ACT_SILU) return mul0(z, rcp_<FAST>(1.0f + exp_<FAST>(-z)));
  return z;
}

template <bool FAST, int ACT> __device__ __forceinline__ float act_slope(float z) {
  if (ACT == GWN_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (ACT == GWN_ACT_GELU) {
    const float e = exp_<FAST>(-0.5f * z * z);
    return normal_cdf<FAST>(z, e) + mul0(0.3989422804f * z, e);
  }
  if (ACT == GWN_ACT_GELU_TANH) {
    const float s = rcp_<FAST>(1.0f + exp_<FAST>(-gelu_u(z)));
    return s + mul0(s * (1.0f - s), z * (1.5957691216f + 0.2140644488f * z * z));
  }
  if (ACT == GWN_ACT_SILU) {
    const float s = rcp_<FAST>(1.0f + exp_<FAST>(-z));
    return mul0(s, 1.0f + mul0(z, 1.0f - s));
  }
  return 1.0f;
}

// v[j] = act(v[j]), the choice made once for the V
template <bool FAST, int ACT, int V> __device__ __forceinline__ void act_all(float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = act_value<FAST, ACT>(v[j]);
}
template <bool FAST, int V> __device__ __forceinline__ void act_vec(float (&v)[V], int act) {
  if (act == GWN_ACT_RELU) act_all<FAST, GWN_ACT_RELU, V>(v);
  if (act == GWN_ACT_GELU) act_all<FAST, GWN_ACT_GELU, V>(v);
  if (act == GWN_ACT_GELU_TANH) act_all<FAST, GWN_ACT_GELU_TANH, V>(v);
  if (act == GWN_ACT_SILU) act_all<FAST, GWN_ACT_SILU, V>(v);
}

// ---- sums ------------------------------------------------------------------------------------
// Partial sums are added pairwise, N values STEP floats apart by log2(N) additions each: one after the other
// they would be the longest chain of a parameter's gradient, and its largest error.
template <int N, int STEP> __device__ __forceinline__ float pair_sum(const float* v) {
  if constexpr (N == 1) return v[0];
  else return pair_sum<N / 2, STEP>(v) + pair_sum<N / 2, STEP>(v + N / 2 * STEP);
}
// of 32 lanes of parts, lane `first`: 8 of its parts at a time pairwise, their sums as they come.  Up to 1024 parts take
// 3 + 4 additions in a chain and the lanes 5 more (32 and 32 before; 172224 rows' gradient 1.8e-7 -> 1.2e-7 off).
__device__ __forceinline__ float part_sum(const float* part, long step, int first, int parts) {
  float sum = 0.0f;
  for (int q = first; q < parts; q += 256) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = q + 32 * j < parts ? part[(q + 32 * j) * step] : 0.0f;
    sum += pair_sum<8, 1>(v);
  }
  return sum;
}

template <typename T> constexpr bool is16 = sizeof(T) == 2;

inline int elem_bytes(int e) { return e == GWN_ELEM_F32 ? 4 : 2; }
inline bool elem_ok(int e) { return e == GWN_ELEM_F32 || e == GWN_ELEM_F16 || e == GWN_ELEM_BF16; }

// p in [0, 1] -> the kernel's threshold and scale
inline Drop drop_of(const unsigned long long* seed_ptr, unsigned long long salt, double p) {
  Drop d{seed_ptr, salt, 0u, 1.0f};
  const double t = p * 16777216.0;
  d.thr = (unsigned)t;
  if ((double)d.thr < t) ++d.thr;
  d.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
  return d;
}

}  // namespace elem
