// y = residual + D(act(x w^T + bias)) in one launch, and its gradients.
//
//   z = x w^T + b,  y = r + D(act(z));  dz = D'(dy) act'(z),  db = sum_m dz,  dx = dz w,  dw = dz^T x
//
// All three products are one tile kernel whose operands lie either with the contraction contiguous
// ("K rows": x and w forward, dz for dx) or with the other index contiguous ("M rows": w for dx, dz
// and x for dw), so that nothing is transposed in memory.
#include "elem.h"

using namespace elem;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// ---- epilogue -----------------------------------------------------------------------------------

// the saved pre-activation: float beside f32 elements, else f16
template <typename T> struct ZType { typedef f16 type; };
template <> struct ZType<float> { typedef float type; };

// Past f16's range it is an infinity, where the derivatives have their limits; relu's border comes out
// of the rounded value as out of the exact one if a positive value stays positive.
__device__ __forceinline__ float z_of(float z, int, float) { return z; }
__device__ __forceinline__ f16 z_of(float z, int act, f16) {
  const f16 h = (f16)z;
  return act == GWN_ACT_RELU && z > 0.0f && h == (f16)0.0f ? (f16)5.9604645e-8f : h;
}

struct Epi {
  const void* bias;
  const void* res; long ld_res;
  void* z; long ldz;
  void* y; long ldy;
  int N, act;
  Drop drop;
  unsigned long long first;  // position of row 0's first element in the mask
};

template <typename T, int V>
__device__ __forceinline__ void load_f(float (&o)[V], const T* p, int rem) {
  if (rem >= V) {
    const Pack<T, V> a = load<T, V>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = (float)a.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = j < rem ? (float)p[j] : 0.0f;
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_f(T* p, const float (&v)[V], int rem) {
  if (rem >= V) {
    Pack<T, V> a;
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = (T)v[j];
    store<T, V>(p, a);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < rem) p[j] = (T)v[j];
  }
}

// an epilogue that computes
bool full(const Epi& e) { return e.act != GWN_ACT_NONE || e.drop.thr; }

// the mask on elements i .. i + V - 1
template <int V>
__device__ __forceinline__ void drop_vec(float (&v)[V], DropKey& key, const Drop& d, unsigned long long i) {
  key.seek(i);
  bool keep[V];
#pragma unroll
  for (int j = 0; j < V; ++j) keep[j] = key.keep((unsigned)i + j, d.thr);
  if ((unsigned)i > 0xFFFFFFFFu - V) {  // the high half steps within
    const unsigned first = (unsigned)i;
    key.rekey(key.hi + 1);
#pragma unroll
    for (int j = 1; j < V; ++j)
      if (first + j < first) keep[j] = key.keep(first + j, d.thr);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = keep[j] ? v[j] * d.scale : 0.0f;
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_part(const T* p, int rem) {
  if (rem >= V) return load<T, V>(p);
  Pack<T, V> a;
#pragma unroll
  for (int j = 0; j < V; ++j) a.v[j] = j < rem ? p[j] : (T)0.0f;
  return a;
}

// V columns n .. of row m, of which `rem` lie within N: all of the epilogue before the residual; b is the
// bias's piece
template <typename T, int V>
__device__ __forceinline__ void before_residual(const Epi& e, DropKey& key, long m, int n, int rem, float (&v)[V],
                                                const Pack<T, V>& b) {
  typedef typename ZType<T>::type Z;
  if (e.bias)
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += (float)b.v[j];
  if (e.z) {
    Z* z = (Z*)e.z + m * e.ldz + n;
    Pack<Z, V> a;
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = z_of(v[j], e.act, Z());
    if (rem >= V) {
      store<Z, V>(z, a);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < rem) z[j] = a.v[j];
    }
  }
  act_vec<is16<T>, V>(v, e.act);
  if (e.drop.thr) drop_vec<V>(v, key, e.drop, e.first + (unsigned long long)m * e.N + n);
}
template <typename T, int V>
__device__ __forceinline__ void epilogue(const Epi& e, DropKey& key, long m, int n, int rem, float (&v)[V]) {
  Pack<T, V> b, r;
  if (e.bias) b = load_part<T, V>((const T*)e.bias + n, rem);
  if (e.res) r = load_part<T, V>((const T*)e.res + m * e.ld_res + n, rem);
  before_residual<T, V>(e, key, m, n, rem, v, b);
  if (e.res)
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += (float)r.v[j];
  store_f<T, V>((T*)e.y + m * e.ldy + n, v, rem);
}

template <int I> struct Int { static constexpr int value = I; };

// ---- the tile kernel ------------------------------------------------------------------------------
//
// A workgroup computes BM x BN of C(m, n) = sum_k A(m, k) B(n, k) by v_mfma_f32_32x32x16 (16-bit) or
// v_mfma_f32_32x32x2_f32, each wave WTM x WTN of it in accumulators.  128 bytes of the contraction a
// step are staged in LDS by buffer loads that write LDS themselves, 16 bytes a lane, in two
// buffers: a step's loads are in flight while the step before is multiplied.  LDS is written
// linearly, so the swizzle that keeps the fragment reads off each other's banks is in the global
// address (swizzle, swizzle_m).  M rows of 16-bit values are read by ds_read_b64_tr_b16, which hands each
// lane four k of its own column.  What lies outside
// the matrices is a load past its buffer resource, which gives zeros.
// Measured (bf16, one launch): 8192^3 842-863 us = 1270-1306 TFLOP/s (a library product of the same operands
// 1510-1560), matrix units busy 71-73% of the cycles (the library's 93%); 20800 x 2048 -> 8192 612-630 us, the units
// busy 65% (the library 535-640 us, 74%), with gelu and z 727-737 us = 947 TFLOP/s.  With the loads in one burst behind the barrier and K rows
// swizzled by row & 7 (half of the LDS cycles conflicts) 8192^3 took 899 us; 64 bytes of k in 4 or 5
// buffers 920, 128 x 256 tiles two a compute unit 1069, 4 waves of 128 x 128 810 but 10% more with an
// epilogue; fragment reads between the products, and wave priorities, changed nothing.
// An operand needs 16-byte aligned rows of whole 16-byte pieces; others are copied to such rows first.

enum { K_ROWS = 0, M_ROWS = 1 };
constexpr int BB = 128, PIECES = BB / 16, PARTS = BB / 32;  // bytes of k a step, its loads and its parts a row
constexpr unsigned OOR = 0x7ffffff0u;  // past every resource
constexpr long MAX_LD = 1 << 20;       // rows further apart are copied: offsets within a tile fit 31 bits

struct Operand {
  const void* p; long ld;
};
struct Gemm {
  Operand a, b;
  int M, N, K, krows;  // krows: the contraction's rows that M-row operands have (K may count padding)
  int tiles_m, tiles_n, splits, kchunk;
  float* part;  // [splits][M][N] (splits > 1)
  Epi e;
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4 rsrc(const void* base, unsigned bytes) {
  const unsigned long long b = (unsigned long long)base;
  return u32x4{(unsigned)b, (unsigned)(b >> 32) & 0xffffu, bytes, 0x00020000u};
}

// 16 bytes a lane from `off` of the resource to LDS at `lds` + 16 lane.  In assembly because the
// compiler waits for every such load before the next transposed LDS read, whichever buffer either
// touches; nothing is written to registers, and the loop below waits for vmcnt itself.
// m0 needs one state before the load; five pass after the assembly begins, since the compiler does not look into it
// for the five that a vector instruction's scalar result (a reloaded spill) needs before a load takes it.
// m0 is reserved, and the compiler refuses it as a clobber: it sets it before each use of its own, and has
// none in this kernel.
__device__ __forceinline__ void load_lds(u32x4 rs, unsigned off, unsigned lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 3\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(lds), "v"(off), "s"(rs)
      : "memory");
}

// where in a K row piece 0 lies: the 16 rows that one LDS cycle reads together (256 bytes; lanes 0-3,
// 12-15, 20-27 and the rest) fall on different banks
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

// the same for an M row of 16-bit values, read 4 rows x 32 columns at a time
template <typename T, int R> __device__ __forceinline__ int swizzle_m(int k) {
  return sizeof(T) == 4 ? 0 : R >= 128 ? (k & 3) << 2 : R == 64 ? (k & 2) << 1 : 0;
}

// R rows (or columns) of an operand, one step of k, by NT threads
template <typename T, int L, int R, int NT>
struct Stage {
  static constexpr int E = 16 / (int)sizeof(T), BK = BB / (int)sizeof(T);
  static constexpr int PER = R * PIECES / NT, CPR = R * (int)sizeof(T) / 16;
  static_assert(R * PIECES % NT == 0 && NT / PIECES % 16 == 0, "whole loads");
  unsigned off[PER];
  int k;  // K rows: this thread's k within a step
  __device__ __forceinline__ void init(const Operand& o, int r0, int rows) {
    const int tid = threadIdx.x;
    const unsigned ldb = (unsigned)(o.ld * (long)sizeof(T));
    if (L == K_ROWS) {
      const int c = (tid % PIECES) ^ swizzle(tid / PIECES);
      k = c * E;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int r = i * (NT / PIECES) + tid / PIECES;
        off[i] = r0 + r < rows ? r * ldb + c * 16 : OOR;
      }
    } else {
      k = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int q = i * NT + tid, kk = q / CPR;
        const int c = (q % CPR) ^ swizzle_m<T, R>(kk);
        off[i] = r0 + c * E < rows ? kk * ldb + c * 16 : OOR;
      }
    }
  }
  // step k0 .. of this operand (kend: the contraction's end, past it all loads are zeros): its
  // resource, then the loads one by one.  A tile's bytes fit 31 bits (MAX_LD).
  u32x4 rs;
  bool ok;
  __device__ __forceinline__ void seek(const Operand& o, int r0, int rows, int k0, int kend, int krows) {
    const unsigned ldb = (unsigned)o.ld * (unsigned)sizeof(T);
    ok = true;
    if (L == K_ROWS) {
      const int nr = rows - r0 < R ? rows - r0 : R;
      ok = k0 + k < kend;
      rs = rsrc((const T*)o.p + (long)r0 * o.ld + k0,
                k0 < kend ? (unsigned)(nr - 1) * ldb + (unsigned)(kend - k0) * (unsigned)sizeof(T) : 0u);
    } else {
      const int left = (kend < krows ? kend : krows) - k0, nk = left < BK ? left : BK;
      rs = rsrc((const T*)o.p + (long)k0 * o.ld + r0,
                nk > 0 ? (unsigned)(nk - 1) * ldb + (unsigned)((rows - r0 + E - 1) / E) * 16u : 0u);
    }
  }
  __device__ __forceinline__ void load(int i, unsigned to, int wave) const {
    load_lds(rs, ok ? off[i] : OOR, to + (i * NT + wave * 64) * 16);
  }
};

// Fragments.  16-bit: the 16 contraction values of quarter ks of a step for one 32-row tile, 8 a
// lane; f32: 8 values, 4 a lane (k = 4 (2 ks + lane / 32) + 0 .. 3), for 4 products of 2.
template <typename T> struct Frag { typedef s16x8 type; };
template <> struct Frag<float> { typedef f32x4 type; };

template <typename T, int L, int R>
__device__ __forceinline__ typename Frag<T>::type frag(const char* s, int row0, int ks, int lane) {
  const int row = row0 + (lane & 31), c = ks * 2 + (lane >> 5);
  if constexpr (L == K_ROWS) {
    return *(const typename Frag<T>::type*)(s + row * BB + ((c ^ swizzle(lane & 31)) << 4));
  } else if constexpr (sizeof(T) == 2) {
    const int i = lane & 15, k = ks * 16 + (lane >> 5) * 8 + (i >> 2);
    const int col = row0 + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
    const char* at = s + k * (R * 2) + (((col >> 3) ^ swizzle_m<T, R>(k)) << 4) + (col & 7) * 2;
    typedef __attribute__((address_space(3))) s16x4* tr_ptr;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 4 * R * 2));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = *(const float*)(s + (c * 4 + e) * (R * 4) + row * 4);
    return v;
  }
}

__device__ __forceinline__ f32x16 mma(s16x8 a, s16x8 b, f32x16 c, bf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
__device__ __forceinline__ f32x16 mma(s16x8 a, s16x8 b, f32x16 c, f16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// workgroup -> (tile, split).  Consecutive workgroups go to the 8 XCDs in turn: each XCD gets a
// contiguous run of tiles, 4 rows of tiles walked column by column, so that its L2 holds the operands
// they share (2 to 16 rows measure within 5%).
__device__ __forceinline__ void place(const Gemm& p, int& tm, int& tn, int& split) {
  const int total = gridDim.x, per = total >> 3;
  int id = blockIdx.x;
  if (id < per * 8) id = (id & 7) * per + (id >> 3);
  const int tiles = p.tiles_m * p.tiles_n;
  split = id / tiles;
  id -= split * tiles;
  const int width = 4 * p.tiles_n, g = id / width, first = g * 4;
  const int rows = p.tiles_m - first < 4 ? p.tiles_m - first : 4;
  id -= g * width;
  tn = id / rows;
  tm = first + id - tn * rows;
}

// ONE: the contraction is one step at most.  Nothing is left to load while it is multiplied, so there is one
// buffer: more workgroups fit a compute unit (f32: 8 of 128x32 for 4; 16-bit: 5 of 128x64 for 3, by their
// registers) and hide each other's loads and stores.  158976 x 224 x 32, the best tile of each: bf16 32.5 -> 20.8
// us, f32 47.6 -> 40.8; 158976 x 32 x 32: 7.8 -> 5.9 and 12.0 -> 9.7.  256x256 fits once either way: no such form.
template <typename T, int LA, int LB, int BM, int BN, int WGM, int WGN, bool ONE>
__global__ __launch_bounds__(64 * WGM * WGN) void gemm_kernel(const Gemm p) {
  constexpr int NT = 64 * WGM * WGN, WTM = BM / WGM, WTN = BN / WGN, TM = WTM / 32, TN = WTN / 32;
  constexpr int BK = BB / (int)sizeof(T), STAGE = (BM + BN) * BB;
  constexpr int EW = WTN + 4;  // floats a row of the epilogue's image of one wave's 32 rows
  constexpr int BUFS = (ONE ? 1 : 2) * STAGE, IMAGES = WGM * WGN * 32 * EW * 4, SMEM = BUFS > IMAGES ? BUFS : IMAGES;
  __shared__ __attribute__((aligned(1024))) char smem[SMEM];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WGM, wn = wave / WGM;
  const unsigned lds0 = (unsigned)(size_t)(lds_ptr_t)smem;
  int tm, tn, split;
  place(p, tm, tn, split);
  const int m0 = tm * BM, n0 = tn * BN;
  const int kbeg = split * p.kchunk, kend = p.K - kbeg < p.kchunk ? p.K : kbeg + p.kchunk;

  Stage<T, LA, BM, NT> sa;
  Stage<T, LB, BN, NT> sb;
  sa.init(p.a, m0, p.M);
  sb.init(p.b, n0, p.N);

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  constexpr int LOADS = sa.PER + sb.PER;
  auto seek = [&](int k0) {
    sa.seek(p.a, m0, p.M, k0, kend, p.krows);
    sb.seek(p.b, n0, p.N, k0, kend, p.krows);
  };
  auto issue = [&](int i, int buf) {
    if (i < sa.PER)
      sa.load(i, lds0 + buf * STAGE, wave);
    else
      sb.load(i - sa.PER, lds0 + buf * STAGE + BM * BB, wave);
  };
  typename Frag<T>::type fa[2][TM], fb[2][TN];
  auto read = [&](int buf, int ks) {
    const char* A = smem + buf * STAGE;
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[ks & 1][i] = frag<T, LA, BM>(A, wm * WTM + i * 32, ks, lane);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[ks & 1][j] = frag<T, LB, BN>(A + BM * BB, wn * WTN + j * 32, ks, lane);
  };
  // A part's products (32 bytes of k).  The step's loads go between those of its first two parts:
  // all at once they would keep the wave from its products until the address unit has taken the
  // whole workgroup's, 16 cycles each.
  constexpr int MM = TM * TN * (sizeof(T) == 2 ? 1 : 4);
  auto multiply = [&](int ks, int part, int to) {
#pragma unroll
    for (int q = 0; q < MM; ++q) {
      const int e = q / (TM * TN), i = q % (TM * TN) / TN, j = q % TN;
      if constexpr (sizeof(T) == 2)
        acc[i][j] = mma(fa[ks & 1][i], fb[ks & 1][j], acc[i][j], T());
      else
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[ks & 1][i][e], fb[ks & 1][j][e], acc[i][j], 0, 0, 0);
      // loads l with l / LOADS < (part MM + q + 1) / (2 MM)
      if (part < 2) {
        const int done = (part * MM + q) * LOADS / (2 * MM), next = (part * MM + q + 1) * LOADS / (2 * MM);
        if (next > done) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int l = done; l < next; ++l) issue(l, to);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  // Two buffers: while one is multiplied the next step is in flight.  A step's last part is multiplied
  // behind the barrier that ends it: by then all its fragments are in registers, so its buffer is free
  // for the loads of the step after next, and the next step's first fragments arrive under those
  // products.
  auto turn = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (ONE && kbeg < kend) {
    seek(kbeg);
#pragma unroll
    for (int l = 0; l < LOADS; ++l) issue(l, 0);
    turn();
    read(0, 0);
#pragma unroll
    for (int ks = 0; ks < PARTS; ++ks) {
      if (ks + 1 < PARTS) read(0, ks + 1);
      multiply(ks, 2, 0);
    }
  } else if (kbeg < kend) {
    seek(kbeg);
#pragma unroll
    for (int l = 0; l < LOADS; ++l) issue(l, 0);
    turn();
    read(0, 0);
    seek(kbeg + BK);
#pragma unroll
    for (int l = 0; l < LOADS / 2; ++l) issue(l, 1);
    int buf = 0;
    for (int k0 = kbeg; k0 < kend; k0 += BK, buf ^= 1) {
#pragma unroll
      for (int ks = 0; ks < PARTS - 1; ++ks) {
        read(buf, ks + 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(ks, ks + 1, buf ^ 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      turn();
      read(buf ^ 1, 0);  // past the last step: zeros, not used
      seek(k0 + 2 * BK);
      __builtin_amdgcn_sched_barrier(0);
      multiply(PARTS - 1, 0, buf);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // the loads past the end write LDS too: vmcnt(0)
  }

  // 32 rows of a wave at a time through LDS, from the accumulators' layout to whole row pieces.  A wait for
  // a load is a wait for all stores before it too, so the bias is read once, and a piece's residual of the
  // next 32 rows before this one's are stored; blocks at the edges read both as they go.  20800 x 2048 ->
  // 8192 in f16: 666 -> 641 us with a bias, 829 -> 673 with a residual too, 991 -> 846 with gelu, dropout and z.
  // Four blocks share their code (unrolled it runs cold through the instruction cache: 720 us with a
  // bias); two are unrolled (158976 x 32 -> 224: 28 -> 22 us).
  constexpr int V = 16 / (int)sizeof(T), LPR = WTN / V, RPI = 64 / LPR, PIECES = 32 / RPI;
  constexpr int ROLL = TM == 4 ? 1 : TM;
  const int n = n0 + wn * WTN + (lane % LPR) * V, rem = p.N - n, mw = m0 + wm * WTM;
  const bool inside = p.splits == 1 && n0 + (wn + 1) * WTN <= p.N;
  Pack<T, V> bias, res[PIECES];
  auto fetch = [&](int q, int row) {
    res[q] = load<T, V>((const T*)p.e.res + (long)(row + q * RPI + lane / LPR) * p.e.ld_res + n);
  };
  if (inside && p.e.bias) bias = load<T, V>((const T*)p.e.bias + n);
  if (inside && p.e.res && mw + 32 <= p.M)
#pragma unroll
    for (int q = 0; q < PIECES; ++q) fetch(q, mw);
  __syncthreads();
  float* img = (float*)smem + wave * 32 * EW;
  DropKey key;
  if (p.e.drop.thr) key.init(p.e.drop, p.e.first + (unsigned long long)m0 * p.N + n0);
#pragma unroll ROLL
  for (int i = 0; i < TM; ++i) {
    const int mi = mw + i * 32;
    auto image = [&](auto I) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          img[((r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * EW + j * 32 + (lane & 31)] = acc[decltype(I)::value][j][r];
    };
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    static_assert(TM == 1 || TM == 2 || TM == 4, "blocks");
    if (TM == 1 || i == 0) image(Int<0>());
    if (TM > 1 && i == 1) image(Int<1 % TM>());
    if (TM > 2 && i == 2) image(Int<2 % TM>());
    if (TM > 2 && i == 3) image(Int<3 % TM>());
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    auto piece = [&](int q, float (&v)[V]) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = img[(q * RPI + lane / LPR) * EW + (lane % LPR) * V + j];
    };
    if (inside && mi + 32 <= p.M) {
      const int next = i + 1 < TM && mi + 64 <= p.M ? mi + 32 : mi;  // these rows again where none follow
#pragma unroll
      for (int q = 0; q < PIECES; ++q) {
        float v[V];
        piece(q, v);
        before_residual<T, V>(p.e, key, mi + q * RPI + lane / LPR, n, V, v, bias);
        if (p.e.res) {
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] += (float)res[q].v[j];
          if (TM == 4 || i + 1 < TM) fetch(q, next);
        }
        store_f<T, V>((T*)p.e.y + (long)(mi + q * RPI + lane / LPR) * p.e.ldy + n, v, V);
      }
    } else {
#pragma unroll 1
      for (int q = 0; q < PIECES; ++q) {
        const long m = mi + q * RPI + lane / LPR;
        float v[V];
        piece(q, v);
        if (m < p.M && rem > 0) {
          if (p.splits > 1)
            store_f<float, V>(p.part + ((long)split * p.M + m) * p.N + n, v, rem);
          else
            epilogue<T, V>(p.e, key, m, n, rem, v);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The splits' sums and the epilogue, bound by reading the sums.  256 / TY pieces of 4 columns x TY lanes of
// splits a workgroup: where there are few outputs their many splits are read side by side (32 x 224
// outputs of 226 splits: 33 -> 5 us).  Fixed order: a lane's splits
// as they come, then the lanes.
template <typename T, int TY>
__global__ __launch_bounds__(256) void join_kernel(const float* part, int splits, int M, int N, Epi e) {
  constexpr int V = 4, TX = 256 / TY;
  __shared__ float sums[TY][TX * V];
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const long per = (N + V - 1) / V, total = per * M;
  DropKey key;
  if (e.drop.thr) key.init(e.drop, (unsigned long long)blockIdx.x * TX * V);
  for (long base = (long)blockIdx.x * TX; base < total; base += (long)gridDim.x * TX) {
    const long q = base + tx, m = q / per;
    const int n = (int)(q - m * per) * V, rem = q < total ? N - n : 0;
    const float* at = part + m * N + n;
    float v[V] = {};
#pragma unroll 4
    for (int s = ty; s < splits; s += TY) {
      float o[V];
      load_f<float, V>(o, at + (long)s * M * N, rem);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += o[j];
    }
    if (TY > 1) {
#pragma unroll
      for (int j = 0; j < V; ++j) sums[ty][tx * V + j] = v[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = 0.0f;
      if (ty == 0)
#pragma unroll
        for (int y = 0; y < TY; ++y)
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] += sums[y][tx * V + j];
      __syncthreads();
    }
    if (ty == 0 && rem > 0) epilogue<T, V>(e, key, m, n, rem, v);
  }
}

// ---- few rows -------------------------------------------------------------------------------------
//
// y for at most 16 MT rows of x: bound by reading w once, so w goes from memory straight into
// v_mfma_f32_16x16x32 (16-bit) or 16x16x4 fragments.  A workgroup has 16 columns (w rows), its waves
// split the contraction: 4 loads of 16 bytes a lane, 256 bytes of each w row, are in flight a wave and
// turn, x's pieces come from the caches.  The waves' sums meet in LDS, then the epilogue.  Rows may
// start anywhere and have any length.  1 x 1024 -> 4096: bf16 and f16 4.0 us, f32 6.4 (w read at 2.1 and 2.6 TB/s);
// 16 x 4096 -> 4096 11.7 and 19.5 us (2.9 and 3.5 TB/s); 12 x 1999 -> 1030 7.5 to 8.8 us in all three.
struct Few {
  const void* x; long ldx;
  const void* w; long ldw;
  int M, N, K;
  Epi e;
};

__device__ __forceinline__ f32x4 mma16(Pack<bf16, 8> a, Pack<bf16, 8> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(Pack<f16, 8> a, Pack<f16, 8> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(Pack<float, 4> a, Pack<float, 4> b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], c, 0, 0, 0);
  return c;
}
// a row's values k .. k + V - 1.  Where they would reach over the row's end K, the V values before the
// end, those before k as zeros: the contraction's order does not matter as long as x and w share it
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_end(const T* row, int k, int K) {
  Pack<T, V> a;
  if (K >= V) {
    const int at = k + V <= K ? k : K - V;
    a = load_odd<T, V>(row + at);
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = at + j >= k ? a.v[j] : (T)0.0f;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = k + j < K ? row[k + j] : (T)0.0f;
  }
  return a;
}

template <typename T, int MT, bool ODD>  // ODD: rows that do not start on 4-byte borders
__global__ __launch_bounds__(1024) void few_kernel(const Few p) {
  constexpr int V = Vec<T>::N, KS = 4 * V, U = 4, LD = 20;
  __shared__ __attribute__((aligned(16))) float sums[16][16 * MT][LD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int n0 = blockIdx.x * 16, row = lane & 15, kl = (lane >> 4) * V;
  const T* w = (const T*)p.w + (long)(n0 + row < p.N ? n0 + row : p.N - 1) * p.ldw;
  const T* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = (const T*)p.x + (long)(i * 16 + row < p.M ? i * 16 + row : p.M - 1) * p.ldx;
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int k0 = wave * KS * U; k0 < p.K; k0 += waves * KS * U) {
    Pack<T, V> a[U], b[MT][U];
    if (k0 + KS * U <= p.K) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * KS + kl;
        a[u] = ODD ? load_odd<T, V>(w + k) : load<T, V>(w + k);
#pragma unroll
        for (int i = 0; i < MT; ++i) b[i][u] = ODD ? load_odd<T, V>(x[i] + k) : load<T, V>(x[i] + k);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a[u] = load_end<T, V>(w, k0 + u * KS + kl, p.K);
#pragma unroll
        for (int i = 0; i < MT; ++i) b[i][u] = load_end<T, V>(x[i], k0 + u * KS + kl, p.K);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = mma16(b[i][u], a[u], acc[i]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[wave][i * 16 + (lane >> 4) * 4 + r][row] = acc[i][r];
  __syncthreads();
  DropKey key;
  if (p.e.drop.thr) key.init(p.e.drop, (unsigned long long)n0);
  for (int q = threadIdx.x; q < 16 * MT * 4; q += blockDim.x) {
    const int m = q >> 2, n = n0 + (q & 3) * 4, rem = p.N - n;
    if (m < p.M && rem > 0) {
      float v[4] = {};
      for (int s = 0; s < waves; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += sums[s][m][(q & 3) * 4 + j];
      epilogue<T, 4>(p.e, key, m, n, rem, v);
    }
  }
}

// rows [rows][ld] -> [rows][ldo] with zeros past `cols`: a 16-byte piece a thread (bound by memory)
template <typename T>
__global__ __launch_bounds__(256) void copy_rows_kernel(const T* x, long ld, long rows, int cols, T* o, int ldo) {
  constexpr int V = Vec<T>::N;
  const int per = ldo / V;
  const long total = rows * per;
  for (long q = (long)blockIdx.x * 256 + threadIdx.x; q < total; q += (long)gridDim.x * 256) {
    const long m = q / per;
    const int n = (int)(q - m * per) * V, rem = cols - n;
    Pack<T, V> a;
    if (rem >= V) {
      a = load<T, V>(x + m * ld + n);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) a.v[j] = j < rem ? x[m * ld + n + j] : (T)0.0f;
    }
    store<T, V>(o + m * ldo + n, a);
  }
}

// ---- dz and the bias's gradient -------------------------------------------------------------------

struct Dz {
  const void* dy; long ld_dy;
  const void* z; long ldz;
  void* dz; int ld;  // [M][ld], columns past N zero; NULL = not written
  float* part;       // [gridDim.y][N] column sums (one stripe: none), and
  void* db;          // where one stripe's go; both NULL = not wanted
  int M, N, tx, stripe;  // TX = 1 << tx; rows a workgroup
  Drop drop;
};

// TX pieces of 16 bytes of columns x a stripe of rows a workgroup, 256 / TX rows at a time; each
// thread sums its columns in fp32 before dz is rounded: dz feeds 16-bit products, so it has their type.
// Bound by memory: dy and z read, dz written (20800 x 8192 in bf16 with gelu: 192 us, 5.3 TB/s; 210 with the
// loads of two rows after the stores of the two before, more with one row's loads in flight).
template <typename T, int ACT>
__global__ __launch_bounds__(256) void dz_kernel(const Dz p) {
  typedef typename ZType<T>::type Z;
  constexpr int V = Vec<T>::N;
  const int TX = 1 << p.tx, TY = 256 >> p.tx;
  __shared__ float cols[256 * V];  // [TY][TX * V]
  const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x >> p.tx;
  const long n = ((long)blockIdx.x * TX + tx) * V;
  const int rem = (int)(p.N - n < V ? p.N - n : V);
  float sum[V] = {};
  DropKey key;
  if (p.drop.thr) key.init(p.drop, (unsigned long long)blockIdx.y * p.stripe * p.N);
  const long first = (long)blockIdx.y * p.stripe, last = first + p.stripe < p.M ? first + p.stripe : p.M;
  auto row = [&](long r, float (&v)[V], const float (&z)[V]) {
    if (ACT != GWN_ACT_NONE) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= act_slope<is16<T>, ACT>(z[j]);
    }
    // last, so that a dropped element's dz is 0 whatever dy and z hold there
    if (p.drop.thr) drop_vec<V>(v, key, p.drop, (unsigned long long)r * p.N + n);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (j >= rem) v[j] = 0.0f;
      sum[j] += v[j];
    }
  };
  long m = first;
  if (rem == V && p.dz && m + 2 * TY <= last) {
    // two rows at a time, the next two's loads before these are stored: a load waits for the stores before it
    Pack<T, V> dy[2][2];
    Pack<Z, V> zs[2][2];
    auto fetch = [&](long at, int to) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const long r = at + u * TY + ty;
        dy[to][u] = load<T, V>((const T*)p.dy + r * p.ld_dy + n);
        if (ACT != GWN_ACT_NONE) zs[to][u] = load<Z, V>((const Z*)p.z + r * p.ldz + n);
      }
    };
    auto pair = [&](int of) {
      fetch(m + 4 * TY <= last ? m + 2 * TY : m, of ^ 1);  // these again at the end
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float v[V], z[V] = {};
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (float)dy[of][u].v[j];
        if (ACT != GWN_ACT_NONE)
#pragma unroll
          for (int j = 0; j < V; ++j) z[j] = (float)zs[of][u].v[j];
        row(m + u * TY + ty, v, z);
        store_f<T, V>((T*)p.dz + (m + u * TY + ty) * p.ld + n, v, V);
      }
      m += 2 * TY;
    };
    fetch(m, 0);
    for (;;) {
      pair(0);
      if (m + 2 * TY > last) break;
      pair(1);
      if (m + 2 * TY > last) break;
    }
  }
  if (rem > 0)
    for (m += ty; m < last; m += 2 * TY) {
      float v[2][V], z[2][V];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const long r = m + u * TY;
        const int here = r < last ? rem : 0;
        load_f<T, V>(v[u], (const T*)p.dy + r * p.ld_dy + n, here);
        if (ACT != GWN_ACT_NONE) load_f<Z, V>(z[u], (const Z*)p.z + r * p.ldz + n, here);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const long r = m + u * TY;
        if (r >= last) break;
        row(r, v[u], z[u]);
        if (p.dz) store_f<T, V>((T*)p.dz + r * p.ld + n, v[u], V);
      }
    }
  if (!p.db) return;
#pragma unroll
  for (int j = 0; j < V; ++j) cols[threadIdx.x * V + j] = sum[j];
  __syncthreads();
  for (int k = threadIdx.x; k < TX * V; k += 256) {
    const long at = (long)blockIdx.x * TX * V + k;
    if (at < p.N) {
      float v = 0.0f;
      for (int q = 0; q < TY; ++q) v += cols[q * TX * V + k];
      if (gridDim.y == 1)
        ((T*)p.db)[at] = (T)v;
      else
        p.part[(long)blockIdx.y * p.N + at] = v;
    }
  }
}

// the stripes' sums, 32 columns x 32 lanes of stripes a workgroup (4 to 5 us), in part_sum's order
template <typename T>
__global__ __launch_bounds__(1024) void colsum_kernel(const float* part, int nparts, int n, T* out) {
  __shared__ float s[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long k = (long)blockIdx.x * 32 + tx;
  s[ty][tx] = k < n ? part_sum(part + k, n, ty, nparts) : 0.0f;
  __syncthreads();
  if (ty == 0 && k < n) out[k] = (T)pair_sum<32, 33>(&s[0][tx]);
}

// ---- plans ------------------------------------------------------------------------------------------

long up(long v, long to) { return (v + to - 1) / to * to; }
int vec_of(int elem) { return 16 / elem_bytes(elem); }

// whether rows of `cols` values can be staged where they lie
bool stageable(const void* p, long ld, int cols, int elem) {
  const int v = vec_of(elem);
  return ((size_t)p & 15) == 0 && ld % v == 0 && ld <= MAX_LD && cols % v == 0;
}
// floats of a copy with whole pieces a row
long copy_floats(long rows, int cols, int elem) { return up(rows * up(cols, vec_of(elem)) * elem_bytes(elem), 16) / 4; }

// The tile and the number of splits of the contraction, by the time (cycles) that a model of a compute
// unit's share gives them: `at_once` workgroups of a tile fit its LDS and take turns at the matrix
// units, a step of theirs takes the slowest of the products, the loads and the loads' latency; splits
// add the writing and joining of their sums.  The numbers are fitted to 3273 measured times of 26
// shapes' three products, 6 tiles and 1 to 256 splits: the model's choice is 2.3% (16-bit) and 1.5%
// (f32) slower than the fastest measured on average, 14% and 22% at worst.  A product at the wrong end
// of the list loses much more: dw of 158976 x 224 x 32 in f32 takes 3100 us unsplit and 63 us in 256.
struct Tile { int bm, bn, at_once; double rate16, rate32; };  // rates: shares of 4096, 256 operations a cycle
constexpr Tile TILES[] = {{256, 256, 1, 0.66, 0.0}, {128, 128, 2, 0.62, 0.86}, {128, 64, 3, 0.30, 0.88},
                          {64, 64, 5, 0.33, 0.88},  {128, 32, 4, 0.17, 0.82},  {32, 128, 4, 0.24, 0.85}};
struct Cost { double load, latency, fixed, epilogue, full, more, join, join_byte; };
constexpr Cost COST16 = {1.0 / 26, 2300, 200, 0.16, 0.28, 1.6, 16000, 1.0 / 710};
constexpr Cost COST32 = {0, 1400, 0, 0, 0, 1, 3200, 1.0 / 1800};
struct Shape { int tile, tiles_m, tiles_n, splits, kchunk; };

// full_epilogue: with an activation or dropout (a residual's loads hide in any tile).  Weighed as one without, 7
// products in 16 bits are 4 to 6% slower than with the fastest tile on average, 17% at worst; so 2 to 4% and 10%
// (5200 x 512 x 2048 with everything: 39.2 -> 37.1 us).  In f32 the products outlast it.
Shape shape_of(int M, int N, int K, int elem, bool full_epilogue) {
  const bool wide = elem == GWN_ELEM_F32;
  const Cost& co = wide ? COST32 : COST16;
  const int bk = wide ? 32 : 64;
  const long cus = gwn_device_cus(), steps = (K + bk - 1) / bk;
  Shape best{};
  double least = 1e300;
  for (int t = 0; t < 6; ++t) {
    const Tile& c = TILES[t];
    const double rate = wide ? c.rate32 * 256 : c.rate16 * 4096;
    if (rate == 0) continue;
    const long tm = (M + c.bm - 1) / c.bm, tn = (N + c.bn - 1) / c.bn, tiles = tm * tn;
    const double product = 2.0 * c.bm * c.bn * bk / rate, loads = (c.bm + c.bn) * 128 * co.load;
    const double step = product > loads ? product : loads;
    const double fixed = co.fixed + c.bm * c.bn * (full_epilogue ? co.full : co.epilogue);
    long last = 0;
    for (long want = 1; want <= 512; want += (want + 3) / 4) {
      const long chunk = (steps + want - 1) / want, splits = chunk ? (steps + chunk - 1) / chunk : 1;
      if (splits == last) continue;
      last = splits;
      const long share = (tiles * splits + cus - 1) / cus, full = share / c.at_once, rest = share % c.at_once;
      const double all = c.at_once * step, some = rest * step;
      double time = full * ((all > co.latency ? all : co.latency) * chunk + fixed * co.more);
      if (rest) time += (some > co.latency ? some : co.latency) * chunk + fixed;
      // A contraction of one step in 16 bits (one buffer): loads, products and stores follow each other in each
      // workgroup, and as many as fit hide only their latency.  Of 12 measured products this takes the fastest
      // tile or one within 2%, the sum above loses 15% (158976 x 224 x 32, 13248 x 512 x 64); in f32 the
      // sum above does so by itself.
      if (steps == 1 && !wide) time = share * (step + fixed) * (c.at_once < 3 ? 3.0 / c.at_once : 1.0);
      if (splits > 1) time += co.join + 8.0 * M * N * splits * co.join_byte;
      if (time < least) {
        least = time;
        best = {t, (int)tm, (int)tn, (int)splits, (int)(chunk * bk)};
      }
      if (tiles * splits > 4 * cus) break;
    }
  }
  return best;
}
long part_floats(int M, int N, int K, int elem, bool full_epilogue = false) {
  const Shape s = shape_of(M, N, K, elem, full_epilogue);
  return s.splits > 1 ? up((long)s.splits * M * N, 4) : 0;
}

template <typename T, int LA, int LB, int BM, int BN, int WGM, int WGN>
void launch_tile(const Gemm& p, int grid, hipStream_t s) {
  if (p.K <= BB / (int)sizeof(T) && BM < 256)
    gemm_kernel<T, LA, LB, BM, BN, WGM, WGN, BM < 256><<<grid, 64 * WGM * WGN, 0, s>>>(p);
  else
    gemm_kernel<T, LA, LB, BM, BN, WGM, WGN, false><<<grid, 64 * WGM * WGN, 0, s>>>(p);
}
template <typename T, int LA, int LB>
void launch_tiles(const Gemm& p, int tile, int grid, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (tile == 0) launch_tile<T, LA, LB, 256, 256, 2, 4>(p, grid, s);
  if (tile == 1) launch_tile<T, LA, LB, 128, 128, 2, 2>(p, grid, s);
  if (tile == 2) launch_tile<T, LA, LB, 128, 64, 2, 2>(p, grid, s);
  if (tile == 3) launch_tile<T, LA, LB, 64, 64, 2, 2>(p, grid, s);
  if (tile == 4) launch_tile<T, LA, LB, 128, 32, 4, 1>(p, grid, s);
  if (tile == 5) launch_tile<T, LA, LB, 32, 128, 1, 4>(p, grid, s);
}

// Rows of the result beyond a launch's MOST_TILES go in launches of their own: 2^29 rows of up to 32 columns and
// more.  (Half of what a grid of 512 threads a workgroup may hold, and place() counts tiles in 32 bits.)
constexpr long MOST_TILES = 1L << 22;

template <typename T>
int gemm(int la, int lb, Operand a, Operand b, int M, int N, int K, int krows, int elem, Epi e, float* part,
         hipStream_t s) {
  const Shape sh = shape_of(M, N, K, elem, full(e));
  const long most = MOST_TILES / sh.tiles_n;  // tiles_n is at most 2^15; splits only where tiles are few
  for (long t = 0; t < sh.tiles_m; t += most) {
    const int tm = (int)(sh.tiles_m - t < most ? sh.tiles_m - t : most);
    const long r0 = t * TILES[sh.tile].bm, rows = t + most < sh.tiles_m ? most * TILES[sh.tile].bm : M - r0;
    const Operand at{(const T*)a.p + r0 * (la == K_ROWS ? a.ld : 1), a.ld};
    Epi et = e;
    et.y = (T*)e.y + r0 * e.ldy;
    if (e.res) et.res = (const T*)e.res + r0 * e.ld_res;
    if (e.z) et.z = (typename ZType<T>::type*)e.z + r0 * e.ldz;
    et.first = (unsigned long long)r0 * e.N;
    const Gemm p{at, b, (int)rows, N, K, krows, tm, sh.tiles_n, sh.splits, sh.kchunk, part, et};
    const int grid = tm * sh.tiles_n * sh.splits;
    if (la == K_ROWS && lb == K_ROWS)
      launch_tiles<T, K_ROWS, K_ROWS>(p, sh.tile, grid, s);
    else if (la == K_ROWS)
      launch_tiles<T, K_ROWS, M_ROWS>(p, sh.tile, grid, s);
    else
      launch_tiles<T, M_ROWS, M_ROWS>(p, sh.tile, grid, s);
    GWN_CHECK_LAUNCH();
  }
  if (sh.splits > 1) {
    const long pieces = (long)M * ((N + 3) / 4), cus = gwn_device_cus(), most = cus * 16;
    if (pieces >= cus * 256 || sh.splits < 8) {
      const long want = (pieces + 255) / 256;
      join_kernel<T, 1><<<(int)(want < most ? want : most), 256, 0, s>>>(part, sh.splits, M, N, e);
    } else {
      const long want = (pieces + 15) / 16;
      join_kernel<T, 16><<<(int)(want < most ? want : most), 256, 0, s>>>(part, sh.splits, M, N, e);
    }
    GWN_CHECK_LAUNCH();
  }
  return GWN_OK;
}

template <typename T>
int copy_rows(const void* x, long ld, long rows, int cols, float*& at, int elem, Operand& o, hipStream_t s) {
  const int ldo = (int)up(cols, vec_of(elem));
  const long want = (rows * (ldo / vec_of(elem)) + 255) / 256, most = (long)gwn_device_cus() * 16;
  copy_rows_kernel<T><<<(int)(want < most ? want : most), 256, 0, s>>>((const T*)x, ld, rows, cols, (T*)at, ldo);
  GWN_CHECK_LAUNCH();
  o = {at, ldo};
  at += copy_floats(rows, cols, elem);
  return GWN_OK;
}

// Where the few-rows kernel is the faster one.  Its workgroups take 2048 (16-bit) or 1024 (f32) values of
// the contraction a turn and read x again each: 1 x 1024 x 4096 in bf16 4.1 us against the tiles' 7.5, 32 x
// 1024 x 4096 5.8 against 9.1, 16 x 4096 x 4096 11.2 against 13.7; but 16 x 8192 x 512 16.5 against 8.6, 24 x
// 4096 x 2048 13.8 against 11.7, 16 x 4096 x 16384 40 against 31.
bool few_rows(const gwn_linear_args* a) {
  return a->M <= 32 && (long)a->M * a->N <= 131072 && a->K <= (a->M <= 16 ? 4096 : 1024);
}

Epi epi_of(const gwn_linear_args* a) {
  return {a->bias, a->residual, a->ld_res, a->act == GWN_ACT_NONE ? nullptr : a->z, a->ldz, a->y, a->ldy, a->N, a->act,
          drop_of(a->seed_ptr, a->salt, a->drop_p), 0};
}

long fwd_floats(const gwn_linear_args* a) {
  if (few_rows(a)) return 0;
  long f = part_floats(a->M, a->N, (int)up(a->K, vec_of(a->elem)), a->elem, full(epi_of(a)));
  if (!stageable(a->x, a->ldx, a->K, a->elem)) f += copy_floats(a->M, a->K, a->elem);
  if (!stageable(a->w, a->ldw, a->K, a->elem)) f += copy_floats(a->N, a->K, a->elem);
  return f;
}

template <typename T>
int fwd(const gwn_linear_args* a, hipStream_t s) {
  const Epi e = epi_of(a);
  if (few_rows(a)) {
    const Few p{a->x, a->ldx, a->w, a->ldw, a->M, a->N, a->K, e};
    const int turn = 16 * vec_of(a->elem), turns = (a->K + turn - 1) / turn;  // values a wave takes at once
    const int threads = 64 * (turns < 16 ? turns : 16), grid = (a->N + 15) / 16;
    const bool odd =
        sizeof(T) == 2 && (((size_t)a->x | (size_t)a->w | (size_t)(a->ldx * 2) | (size_t)(a->ldw * 2)) & 3);
    if constexpr (sizeof(T) == 2)
      if (odd) (a->M <= 16 ? few_kernel<T, 1, true> : few_kernel<T, 2, true>)<<<grid, threads, 0, s>>>(p);
    if (!odd) (a->M <= 16 ? few_kernel<T, 1, false> : few_kernel<T, 2, false>)<<<grid, threads, 0, s>>>(p);
    GWN_CHECK_LAUNCH();
    return GWN_OK;
  }
  Operand x{a->x, a->ldx}, w{a->w, a->ldw};
  float* at = a->workspace;
  if (!stageable(a->x, a->ldx, a->K, a->elem)) {
    const int rc = copy_rows<T>(a->x, a->ldx, a->M, a->K, at, a->elem, x, s);
    if (rc) return rc;
  }
  if (!stageable(a->w, a->ldw, a->K, a->elem)) {
    const int rc = copy_rows<T>(a->w, a->ldw, a->N, a->K, at, a->elem, w, s);
    if (rc) return rc;
  }
  const int kp = (int)up(a->K, vec_of(a->elem));  // a copy's zeros included
  return gemm<T>(K_ROWS, K_ROWS, x, w, a->M, a->N, kp, kp, a->elem, e, at, s);
}

struct BwdPlan {
  bool write_dz, copy_x, copy_w;  // dz apart from dy; operands that have to be copied
  int parts, tx, stripe, ld_dz;
  long floats;
};
BwdPlan bwd_plan(const gwn_linear_bwd_args* a) {
  BwdPlan q;
  const int v = vec_of(a->elem);
  const bool product = (a->dx || a->dw) && a->M;
  q.write_dz = product && (a->act != GWN_ACT_NONE || a->drop_p > 0.0 || !stageable(a->dy, a->ld_dy, a->N, a->elem));
  q.copy_x = a->dw && a->M && !stageable(a->x, a->ldx, a->K, a->elem);
  q.copy_w = a->dx && a->M && !stageable(a->w, a->ldw, a->K, a->elem);
  q.ld_dz = (int)up(a->N, v);
  const int pieces = q.ld_dz / v;
  q.tx = pieces <= 8 ? 3 : pieces <= 16 ? 4 : pieces <= 32 ? 5 : 6;
  const long bx = (pieces + (1 << q.tx) - 1) >> q.tx, ty = 256 >> q.tx;
  long parts = (8L * gwn_device_cus() + bx - 1) / bx, most = (a->M + 4 * ty - 1) / (4 * ty);
  if (parts > most) parts = most;
  if (parts > 1024) parts = 1024;
  if (parts < 1 || a->M <= 16 * ty) parts = 1;  // few rows: a launch less
  q.stripe = (int)up((a->M + parts - 1) / parts, 2 * ty);
  q.parts = a->M ? (a->M + q.stripe - 1) / q.stripe : 1;
  q.floats = a->dbias && q.parts > 1 ? up((long)q.parts * a->N, 4) : 0;
  if (q.write_dz) q.floats += copy_floats(a->M, a->N, a->elem);
  if (q.copy_x) q.floats += copy_floats(a->M, a->K, a->elem);
  if (q.copy_w) q.floats += copy_floats(a->N, a->K, a->elem);
  long part = 0;
  if (a->dx && a->M) part = part_floats(a->M, a->K, q.ld_dz, a->elem);
  if (a->dw) {
    const long f = part_floats(a->N, a->K, a->M, a->elem);
    if (f > part) part = f;
  }
  q.floats += part;
  return q;
}

template <typename T>
int bwd(const gwn_linear_bwd_args* a, hipStream_t s) {
  const BwdPlan q = bwd_plan(a);
  const Drop drop = drop_of(a->seed_ptr, a->salt, a->drop_p);
  float* at = a->workspace;
  float* sums = at;
  if (a->dbias && q.parts > 1) at += up((long)q.parts * a->N, 4);
  Operand dz{a->dy, a->ld_dy}, x{a->x, a->ldx}, w{a->w, a->ldw};
  if (q.write_dz) {
    dz = {at, q.ld_dz};
    at += copy_floats(a->M, a->N, a->elem);
  }
  if (q.write_dz || a->dbias) {
    const Dz d{a->dy, a->ld_dy, a->z, a->ldz, q.write_dz ? (void*)dz.p : nullptr, q.ld_dz, sums, a->dbias, a->M,
               a->N, q.tx, q.stripe, drop};
    const dim3 grid((q.ld_dz / vec_of(a->elem) + (1 << q.tx) - 1) >> q.tx, q.parts);
    if (a->act == GWN_ACT_NONE) dz_kernel<T, GWN_ACT_NONE><<<grid, 256, 0, s>>>(d);
    if (a->act == GWN_ACT_RELU) dz_kernel<T, GWN_ACT_RELU><<<grid, 256, 0, s>>>(d);
    if (a->act == GWN_ACT_GELU) dz_kernel<T, GWN_ACT_GELU><<<grid, 256, 0, s>>>(d);
    if (a->act == GWN_ACT_GELU_TANH) dz_kernel<T, GWN_ACT_GELU_TANH><<<grid, 256, 0, s>>>(d);
    if (a->act == GWN_ACT_SILU) dz_kernel<T, GWN_ACT_SILU><<<grid, 256, 0, s>>>(d);
    GWN_CHECK_LAUNCH();
  }
  if (a->dbias && q.parts > 1) {
    colsum_kernel<T><<<(a->N + 31) / 32, 1024, 0, s>>>(sums, q.parts, a->N, (T*)a->dbias);
    GWN_CHECK_LAUNCH();
  }
  int rc = GWN_OK;
  if (q.copy_x && (rc = copy_rows<T>(a->x, a->ldx, a->M, a->K, at, a->elem, x, s))) return rc;
  if (q.copy_w && (rc = copy_rows<T>(a->w, a->ldw, a->N, a->K, at, a->elem, w, s))) return rc;
  Epi e{};
  if (a->dx && a->M) {
    e.y = a->dx, e.ldy = a->ld_dx, e.N = a->K;
    // the contraction over N takes dz's padding in; w has N rows, past them its resource gives zeros
    rc = gemm<T>(K_ROWS, M_ROWS, dz, w, a->M, a->K, q.ld_dz, a->N, a->elem, e, at, s);
    if (rc) return rc;
  }
  if (a->dw) {
    e.y = a->dw, e.ldy = a->ld_dw, e.N = a->K;
    rc = gemm<T>(M_ROWS, M_ROWS, dz, x, a->N, a->K, a->M, a->M, a->elem, e, at, s);
    if (rc) return rc;
  }
  return GWN_OK;
}

long range_bytes(long rows, long ld, long cols, int bytes) { return rows ? ((rows - 1) * ld + cols) * bytes : 0; }

int shape_checks(int M, int N, int K, int elem, int act, double drop_p, const void* seed_ptr) {
  GWN_REQUIRE(elem_ok(elem), "linear: unknown element type");
  GWN_REQUIRE(act >= GWN_ACT_NONE && act <= GWN_ACT_SILU, "linear: unknown activation");
  GWN_REQUIRE(M >= 0 && N > 0 && K > 0, "linear: M must be >= 0, N and K > 0");
  GWN_REQUIRE(M <= (1 << 30) && N <= MAX_LD && K <= MAX_LD, "linear: M is at most 2^30, N and K 2^20");
  GWN_REQUIRE(drop_p >= 0.0 && drop_p <= 1.0, "linear: the dropout rate must be between 0 and 1");
  GWN_REQUIRE(drop_p == 0.0 || (seed_ptr && ((size_t)seed_ptr & 7) == 0), "linear: dropout needs a seed");
  return GWN_OK;
}

}  // namespace

extern "C" {

long gwn_linear_fwd_workspace_floats(const gwn_linear_args* a) {
  if (!a || shape_checks(a->M, a->N, a->K, a->elem, a->act, a->drop_p, a->seed_ptr) || a->M == 0) return 0;
  return fwd_floats(a);
}

int gwn_linear_fwd(const gwn_linear_args* a, hipStream_t stream) {
  GWN_REQUIRE(a, "linear: null arguments");
  const int rc = shape_checks(a->M, a->N, a->K, a->elem, a->act, a->drop_p, a->seed_ptr);
  if (rc) return rc;
  if (a->M == 0) return GWN_OK;
  GWN_REQUIRE(a->x && a->w && a->y, "linear: null pointer");
  GWN_REQUIRE(a->ldx >= a->K && a->ldw >= a->K && a->ldy >= a->N && (!a->residual || a->ld_res >= a->N) &&
                  (!a->z || a->ldz >= a->N),
              "linear: a leading dimension is shorter than the row");
  const int e = elem_bytes(a->elem);
  GWN_REQUIRE((((size_t)a->x | (size_t)a->w | (size_t)a->bias | (size_t)a->residual | (size_t)a->y | (size_t)a->z) &
               (e - 1)) == 0,
              "linear: a pointer is not aligned to its element");
  const long ws = fwd_floats(a);
  GWN_REQUIRE(ws == 0 || (a->workspace && ((size_t)a->workspace & 15) == 0), "linear: the workspace is missing");
  GWN_DEBUG_RANGE(a->x, range_bytes(a->M, a->ldx, a->K, e), "linear x");
  GWN_DEBUG_RANGE(a->w, range_bytes(a->N, a->ldw, a->K, e), "linear w");
  GWN_DEBUG_RANGE(a->residual, range_bytes(a->M, a->ld_res, a->N, e), "linear residual");
  GWN_DEBUG_RANGE(a->y, range_bytes(a->M, a->ldy, a->N, e), "linear y");
  GWN_DEBUG_RANGE(a->z, range_bytes(a->M, a->ldz, a->N, e), "linear z");
  GWN_DEBUG_RANGE(a->workspace, ws * 4, "linear workspace");
  if (a->elem == GWN_ELEM_F32) return fwd<float>(a, stream);
  if (a->elem == GWN_ELEM_F16) return fwd<f16>(a, stream);
  return fwd<bf16>(a, stream);
}

long gwn_linear_bwd_workspace_floats(const gwn_linear_bwd_args* a) {
  if (!a || shape_checks(a->M, a->N, a->K, a->elem, a->act, a->drop_p, a->seed_ptr)) return 0;
  return bwd_plan(a).floats;
}

int gwn_linear_bwd(const gwn_linear_bwd_args* a, hipStream_t stream) {
  GWN_REQUIRE(a, "linear_bwd: null arguments");
  const int rc = shape_checks(a->M, a->N, a->K, a->elem, a->act, a->drop_p, a->seed_ptr);
  if (rc) return rc;
  if (!a->dx && !a->dw && !a->dbias) return GWN_OK;
  GWN_REQUIRE(a->M == 0 || a->dy, "linear_bwd: null pointer");
  GWN_REQUIRE(a->M == 0 || ((!a->dx || a->w) && (!a->dw || a->x) && (a->act == GWN_ACT_NONE || a->z)),
              "linear_bwd: null pointer");
  GWN_REQUIRE(a->M == 0 || (a->ld_dy >= a->N && (!a->dw || a->ldx >= a->K) && (!a->dx || a->ldw >= a->K) &&
                            (a->act == GWN_ACT_NONE || a->ldz >= a->N) && (!a->dx || a->ld_dx >= a->K)),
              "linear_bwd: a leading dimension is shorter than the row");
  GWN_REQUIRE(!a->dw || a->ld_dw >= a->K, "linear_bwd: a leading dimension is shorter than the row");
  const int e = elem_bytes(a->elem);
  GWN_REQUIRE((((size_t)a->dy | (size_t)a->x | (size_t)a->w | (size_t)a->z | (size_t)a->dx | (size_t)a->dw |
                (size_t)a->dbias) & (e - 1)) == 0,
              "linear_bwd: a pointer is not aligned to its element");
  const long ws = bwd_plan(a).floats;
  GWN_REQUIRE(ws == 0 || (a->workspace && ((size_t)a->workspace & 15) == 0), "linear_bwd: the workspace is missing");
  GWN_DEBUG_RANGE(a->dy, range_bytes(a->M, a->ld_dy, a->N, e), "linear_bwd dy");
  if (a->dw) GWN_DEBUG_RANGE(a->x, range_bytes(a->M, a->ldx, a->K, e), "linear_bwd x");
  if (a->dx) GWN_DEBUG_RANGE(a->w, range_bytes(a->N, a->ldw, a->K, e), "linear_bwd w");
  if (a->act != GWN_ACT_NONE)
    GWN_DEBUG_RANGE(a->z, range_bytes(a->M, a->ldz, a->N, a->elem == GWN_ELEM_F32 ? 4 : 2), "linear_bwd z");
  GWN_DEBUG_RANGE(a->dx, range_bytes(a->M, a->ld_dx, a->K, e), "linear_bwd dx");
  GWN_DEBUG_RANGE(a->dw, range_bytes(a->N, a->ld_dw, a->K, e), "linear_bwd dw");
  GWN_DEBUG_RANGE(a->workspace, ws * 4, "linear_bwd workspace");
  if (a->elem == GWN_ELEM_F32) return bwd<float>(a, stream);
  if (a->elem == GWN_ELEM_F16) return bwd<f16>(a, stream);
  return bwd<bf16>(a, stream);
}

}  // extern "C"
