// Layer norm over the last axis, forward and backward.
//
//   mean = sum x / C,  rstd = (sum (x - mean)^2 / C + eps)^(-1/2),  y = (x - mean) rstd g + b
//   xh = (x - mean) rstd,  h = dy g,  dx = rstd (h - sum(h) / C - xh sum(h xh) / C)
//   dg = sum_rows dy xh,  db = sum_rows dy
//
// Bound by memory: x read and y written once forward; x and dy read, dx written once backward.  A
// row lives in the registers of a group of G lanes (G = 4 .. 64 lanes of a wave, or a workgroup of as
// many waves as its 16-byte vectors need), one vector a lane, so that the variance is the centred sum of squares and
// nothing is read twice.  The centred values' own mean is taken off again (the corrected two-pass
// form): the first mean's rounding, which 1 / sqrt(eps) would magnify in a row that hardly varies,
// drops out, and a constant row gives exactly b.  Groups walk the rows; each lane keeps its columns' sums of dg and db in
// registers over all rows its group sees, a workgroup adds its groups up and writes one partial row,
// and a second launch adds the partial rows in a fixed order.  Rows longer than a workgroup's
// registers are looped over (they stay in the L2 cache between the passes).
//
// Measured, 20800 x 4096 in bf16: forward 67-71 us, backward 98 us + 4 us for the partial rows, 5.0 and 5.2
// TB/s, as a large copy.  Over widths (170 MB of x, forward and backward): rows of 32 to 8192 channels that fill their waves
// with whole vectors run at 4.5 to 5.3 TB/s; others of these widths at 2.9 to 5.1 (idle lanes, unaligned pieces), and 16-bit
// rows up to 16384 at 3.5 to 4.4.  Short rows in 16 bits leave lanes of the smallest group idle: 0.8 / 1.6 TB/s at 5
// channels, 1.9 / 3.0 at 8, 2.4 / 2.2 at 12 (f32 2.8 to 5.0).  Looped rows (f32 from 8193 channels, 16 bits from 16385) take 1.8 to 3.2.
// Several vectors a lane took the backward's
// registers and with them the waves that hide its latency: 195 us with two.
#include "elem.h"

using namespace elem;

namespace {

constexpr int THREADS = 256, MOST = 1024;  // a workgroup's, of small groups and at most

struct LnFwd {
  const void* x; long ldx; long rows; int c;
  const void* gamma; const void* beta; float eps;
  void* y; long ldy; float* mean; float* rstd;
};
struct LnBwd {
  const void* dy; long ld_dy; const void* x; long ldx; long rows; int c;
  const void* gamma; const float* mean; const float* rstd;
  void* dx; long ld_dx; float* part;  // part [grid][2][c], or NULL
};

// V elements at p as floats; the first `rem` of them where the row ends within (others `fill`)
template <typename T, int V>
__device__ __forceinline__ void load_f(float (&o)[V], const T* p, int rem, float fill) {
  if (rem >= V) {
    const Pack<T, V> a = load<T, V>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = (float)a.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = j < rem ? (float)p[j] : fill;
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

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// sum over G lanes of a wave, the same value in all of them: neighbours, pairs, the halves of 8 and of
// 16 by mirrored lane operands, 16s and 32s by shuffles
template <int G> __device__ __forceinline__ float lanes_sum(float v) {
  if (G >= 2) v += dpp<0xB1>(v);
  if (G >= 4) v += dpp<0x4E>(v);
  if (G >= 8) v += dpp<0x141>(v);
  if (G >= 16) v += dpp<0x140>(v);
  if (G >= 32) v += __shfl_xor(v, 16, 64);
  if (G >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}
// Sums over the lanes of a group (G = 0: a workgroup), the same values in all of them.  A workgroup's go
// through `lds`, one barrier: the caller alternates between two areas, so that an area is written again
// only behind the other's barrier, which all its readers have reached.
template <int G, int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float (*lds)[MOST / 64]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = lanes_sum<(G ? G : 64)>(v[k]);
  if (G == 0) {
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) lds[k][threadIdx.x >> 6] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = 0.0f;
      for (int w = 0; w < (int)blockDim.x >> 6; ++w) v[k] += lds[k][w];
    }
  }
}

// A lane's vectors of a row, I of them.  EVEN: the row is whole vectors, lanes past its end have none.
// Otherwise the vector that would reach over the row's end starts V columns before the end, and its
// first cut(i) values, another lane's too, are left out of the sums: no load is predicated by element
// (but in rows shorter than a vector).
template <int V, int G, bool EVEN>
struct Span {
  int c, lane;
  static constexpr bool TINY = !EVEN && G == 4;  // rows shorter than a vector are among these
  __device__ __forceinline__ int whole(int i) const { return (lane + (int)blockDim.x * i) * V; }
  __device__ __forceinline__ bool in(int i) const { return whole(i) < c; }
  __device__ __forceinline__ int at(int i) const {
    const int w = whole(i);
    if (EVEN) return w;
    return TINY && c < V ? 0 : w + V <= c ? w : c - V;
  }
  // whether value j of vector i, which is in the row, is this lane's
  __device__ __forceinline__ bool own(int i, int j) const {
    if (EVEN) return true;
    return TINY && c < V ? j < c : j >= whole(i) - at(i);
  }
  __device__ __forceinline__ bool counts(int i, int j) const { return in(i) && own(i, j); }
  // whether value j of vector i is one of the row's, this lane's or not
  __device__ __forceinline__ bool there(int i, int j) const { return in(i) && !(TINY && c < V && j >= c); }
  // zeros where there is no vector
  template <typename T> __device__ __forceinline__ Pack<T, V> get(const T* row, int i) const {
    Pack<T, V> a{};
    if (TINY && c < V) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (in(i) && j < c) a.v[j] = row[j];
    } else if (in(i)) {
      a = load<T, V>(row + at(i));
    }
    return a;
  }
  template <typename T> __device__ __forceinline__ void put(T* row, int i, const float (&v)[V]) const {
    if (!in(i)) return;
    if (TINY && c < V) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < c) row[j] = (T)v[j];
    } else {
      Pack<T, V> a;
#pragma unroll
      for (int j = 0; j < V; ++j) a.v[j] = (T)v[j];
      store<T, V>(row + at(i), a);
    }
  }
};

// the parameters' vectors as floats (`none` where there are no parameters)
template <typename W, int V, typename S>
__device__ __forceinline__ void params_of(float (&o)[V], const S& sp, const void* p, int i, float none) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = none;
    return;
  }
  const Pack<W, V> a = sp.template get<W>((const W*)p, i);
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = (float)a.v[j];
}

template <typename T, typename W, int G, int I, bool EVEN>
__global__ __launch_bounds__(G ? THREADS : I == 1 ? MOST : MOST / 2) void ln_fwd_kernel(const LnFwd p) {
  constexpr int V = Vec<T>::N, PER = G ? THREADS / (G ? G : 1) : 1;
  static_assert(G == 0 || I == 1, "one vector a lane");
  constexpr bool HOLD = I == 1;  // the parameters stay in registers over the rows
  __shared__ float red[2][2][MOST / 64];
  const Span<V, G, EVEN> sp{p.c, G ? (int)threadIdx.x % (G ? G : 1) : (int)threadIdx.x};
  const float c = (float)p.c;
  const long step = (long)gridDim.x * PER;
  float g[I][V], b[I][V];
  if (HOLD) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      params_of<W, V>(g[i], sp, p.gamma, i, 1.0f);
      params_of<W, V>(b[i], sp, p.beta, i, 0.0f);
    }
  }
  long row = (long)blockIdx.x * PER + (G ? threadIdx.x / (G ? G : 1) : 0);
  Pack<T, V> next[I];
  if (row < p.rows)
#pragma unroll
    for (int i = 0; i < I; ++i) next[i] = sp.template get<T>((const T*)p.x + row * p.ldx, i);
  // whole groups leave together; a whole workgroup where the group is one
  for (; row < p.rows; row += step) {
    float v[I][V], s[1] = {0.0f}, d[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = (float)next[i].v[j];
        s[0] += sp.own(i, j) ? v[i][j] : 0.0f;  // zeros where there is no vector
      }
    if (row + step < p.rows)  // the next row's loads are in flight during this row's sums
#pragma unroll
      for (int i = 0; i < I; ++i) next[i] = sp.template get<T>((const T*)p.x + (row + step) * p.ldx, i);
    group_sums<G, 1>(s, red[0]);
    const float mean = s[0] / c;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] -= mean;
        const float w = sp.counts(i, j) ? v[i][j] : 0.0f;
        d[0] += w;
        d[1] += w * w;
      }
    group_sums<G, 2>(d, red[1]);
    const float left = d[0] / c;
    const float rstd = 1.0f / sqrtf(fmaxf(d[1] / c - left * left, 0.0f) + p.eps);
    if (p.mean && sp.lane == 0) {
      p.mean[row] = mean + left;
      p.rstd[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
      if (!HOLD) {
        params_of<W, V>(g[i], sp, p.gamma, i, 1.0f);
        params_of<W, V>(b[i], sp, p.beta, i, 0.0f);
      }
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = (v[i][j] - left) * rstd * g[i][j] + b[i][j];
      sp.template put<T>((T*)p.y + row * p.ldy, i, o);
    }
  }
}

// one sum over a workgroup
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = lanes_sum<64>(v);
  __syncthreads();  // the last sum's reads are done
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

// rows of any length, a workgroup each: three passes over a row
template <typename T, typename W>
__global__ __launch_bounds__(THREADS) void ln_fwd_long_kernel(const LnFwd p) {
  constexpr int V = Vec<T>::N;
  __shared__ float red[THREADS / 64];
  const float c = (float)p.c;
  for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = (const T*)p.x + row * p.ldx;
    T* y = (T*)p.y + row * p.ldy;
    float sum = 0.0f, sq = 0.0f, sd = 0.0f;
    for (long at = (long)threadIdx.x * V; at < p.c; at += THREADS * V) {
      float v[V];
      load_f<T, V>(v, x + at, (int)(p.c - at), 0.0f);
#pragma unroll
      for (int j = 0; j < V; ++j) sum += v[j];
    }
    const float first = block_sum(sum, red) / c;
    for (long at = (long)threadIdx.x * V; at < p.c; at += THREADS * V) {
      float v[V];
      load_f<T, V>(v, x + at, (int)(p.c - at), first);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[j] - first;
        sq += d * d;
        sd += d;
      }
    }
    const float left = block_sum(sd, red) / c, mean = first + left;
    const float rstd = 1.0f / sqrtf(fmaxf(block_sum(sq, red) / c - left * left, 0.0f) + p.eps);
    if (p.mean && threadIdx.x == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    for (long at = (long)threadIdx.x * V; at < p.c; at += THREADS * V) {
      const int rem = (int)(p.c - at);
      float v[V], g[V], b[V];
      load_f<T, V>(v, x + at, rem, 0.0f);
      if (p.gamma) load_f<W, V>(g, (const W*)p.gamma + at, rem, 0.0f);
      if (p.beta) load_f<W, V>(b, (const W*)p.beta + at, rem, 0.0f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[j] = ((v[j] - first) - left) * rstd;
        if (p.gamma) v[j] *= g[j];
        if (p.beta) v[j] += b[j];
      }
      store_f<T, V>(y + at, v, rem);
    }
  }
}

template <typename T, typename W, int G, int I, bool EVEN>
__global__ __launch_bounds__(G ? THREADS : I == 1 ? MOST : MOST / 2) void ln_bwd_kernel(const LnBwd p) {
  constexpr int V = Vec<T>::N, PER = G ? THREADS / (G ? G : 1) : 1;
  static_assert(G == 0 || I == 1, "one vector a lane");
  constexpr bool HOLD = I == 1;
  __shared__ float red[2][2][MOST / 64];
  __shared__ float cols[PER > 1 ? 2 * G * V : 1];
  const Span<V, G, EVEN> sp{p.c, G ? (int)threadIdx.x % (G ? G : 1) : (int)threadIdx.x};
  const float inv = 1.0f / (float)p.c;
  float dg[I][V] = {}, db[I][V] = {}, g[I][V];
  if (HOLD)
#pragma unroll
    for (int i = 0; i < I; ++i) params_of<W, V>(g[i], sp, p.gamma, i, 1.0f);
  const long step = (long)gridDim.x * PER;
  long row = (long)blockIdx.x * PER + (G ? threadIdx.x / (G ? G : 1) : 0);
  Pack<T, V> nx[I], ny[I];
  float nmean = 0.0f, nrstd = 0.0f;
  auto fetch = [&](long r) {
    nmean = p.mean[r], nrstd = p.rstd[r];
#pragma unroll
    for (int i = 0; i < I; ++i) {
      nx[i] = sp.template get<T>((const T*)p.x + r * p.ldx, i);
      ny[i] = sp.template get<T>((const T*)p.dy + r * p.ld_dy, i);
    }
  };
  if (row < p.rows) fetch(row);
  for (int turn = 0; row < p.rows; row += step, turn ^= 1) {
    const float mean = nmean, rstd = nrstd;
    float v[I][V], h[I][V], s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // 0 where there is none: mean rstd may pass fp32's range, and an infinity by h = 0 is a NaN in the sums
        v[i][j] = ((float)nx[i].v[j] - mean) * (sp.there(i, j) ? rstd : 0.0f);
        h[i][j] = (float)ny[i].v[j];
      }
    if (row + step < p.rows) fetch(row + step);
#pragma unroll
    for (int i = 0; i < I; ++i) {
      if (!HOLD) params_of<W, V>(g[i], sp, p.gamma, i, 1.0f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        dg[i][j] += h[i][j] * v[i][j];  // of a cut vector's first values another lane has the sums
        db[i][j] += h[i][j];
        h[i][j] *= g[i][j];
        const float w = sp.own(i, j) ? h[i][j] : 0.0f;  // zeros where there is no vector
        s[0] += w;
        s[1] += w * v[i][j];
      }
    }
    if (!p.dx) continue;
    group_sums<G, 2>(s, red[turn]);
    const float s1 = s[0] * inv, s2 = s[1] * inv;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = rstd * (h[i][j] - s1 - v[i][j] * s2);
      sp.template put<T>((T*)p.dx + row * p.ld_dx, i, o);
    }
  }
  if (!p.part) return;
  float* part = p.part + (long)blockIdx.x * 2 * p.c;
  if constexpr (PER == 1) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      if (EVEN) {
        sp.template put<float>(part, i, dg[i]);
        sp.template put<float>(part + p.c, i, db[i]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (sp.counts(i, j)) {
            part[sp.at(i) + j] = dg[i][j];
            part[p.c + sp.at(i) + j] = db[i][j];
          }
      }
    }
  } else {
    // a wave's groups by shuffles, then the waves one after the other
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int o = G; o < 64; o <<= 1) {
          dg[i][j] += __shfl_xor(dg[i][j], o, 64);
          db[i][j] += __shfl_xor(db[i][j], o, 64);
        }
    const int wave = threadIdx.x >> 6;
    for (int w = 0; w < THREADS / 64; ++w) {
      __syncthreads();
      if (wave == w && (threadIdx.x & 63) < G) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (sp.counts(i, j)) {
              const int at = sp.at(i) + j;
              cols[at] = w ? cols[at] + dg[i][j] : dg[i][j];
              cols[G * V + at] = w ? cols[G * V + at] + db[i][j] : db[i][j];
            }
      }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < p.c; k += THREADS) {
      part[k] = cols[k];
      part[p.c + k] = cols[G * V + k];
    }
  }
}

// dx of rows of any length, a workgroup each
template <typename T, typename W>
__global__ __launch_bounds__(THREADS) void ln_bwd_long_kernel(const LnBwd p) {
  constexpr int V = Vec<T>::N;
  __shared__ float red[THREADS / 64];
  const float inv = 1.0f / (float)p.c;
  for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = (const T*)p.x + row * p.ldx;
    const T* dy = (const T*)p.dy + row * p.ld_dy;
    T* dx = (T*)p.dx + row * p.ld_dx;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
      for (long at = (long)threadIdx.x * V; at < p.c; at += THREADS * V) {
        const int rem = (int)(p.c - at);
        float v[V], h[V], g[V];
        load_f<T, V>(v, x + at, rem, mean);
        load_f<T, V>(h, dy + at, rem, 0.0f);
        if (p.gamma) load_f<W, V>(g, (const W*)p.gamma + at, rem, 0.0f);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[j] = (v[j] - mean) * rstd;
          if (p.gamma) h[j] *= g[j];
        }
        if (pass == 0) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            s1 += h[j];
            s2 += h[j] * v[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = rstd * (h[j] - s1 - v[j] * s2);
          store_f<T, V>(dx + at, v, rem);
        }
      }
      if (pass == 0) {
        s1 = block_sum(s1, red) * inv;
        s2 = block_sum(s2, red) * inv;
      }
    }
  }
}

// partial dg / db of rows of any length: 64 vectors of columns x 4 rows a workgroup, rows split
// over gridDim.y
template <typename T>
__global__ __launch_bounds__(THREADS) void ln_cols_long_kernel(const LnBwd p) {
  constexpr int V = Vec<T>::N;
  __shared__ float cols[4][2][64 * V];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const long at = ((long)blockIdx.x * 64 + tx) * V;
  const int rem = (int)(p.c - at < V ? p.c - at : V);
  float dg[V] = {}, db[V] = {};
  if (rem > 0)
    for (long row = (long)blockIdx.y * 4 + ty; row < p.rows; row += (long)gridDim.y * 4) {
      float v[V], h[V];
      load_f<T, V>(v, (const T*)p.x + row * p.ldx + at, rem, 0.0f);
      load_f<T, V>(h, (const T*)p.dy + row * p.ld_dy + at, rem, 0.0f);
      const float mean = p.mean[row], rstd = p.rstd[row];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        dg[j] += h[j] * ((v[j] - mean) * rstd);
        db[j] += h[j];
      }
    }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    cols[ty][0][tx * V + j] = dg[j];
    cols[ty][1][tx * V + j] = db[j];
  }
  __syncthreads();
  float* part = p.part + (long)blockIdx.y * 2 * p.c;
  for (int k = threadIdx.x; k < 64 * V; k += THREADS) {
    const long col = (long)blockIdx.x * 64 * V + k;
    if (col < p.c) {
      part[col] = cols[0][0][k] + cols[1][0][k] + cols[2][0][k] + cols[3][0][k];
      part[p.c + col] = cols[0][1][k] + cols[1][1][k] + cols[2][1][k] + cols[3][1][k];
    }
  }
}

// out[k] = sum over parts of part[.][k]: 32 columns x 32 lanes of parts a workgroup, in part_sum's order.  The
// workgroups walk the columns: a grid has fewer than 2^32 threads, and columns go up to 2^31.
constexpr long REDUCE_GRID = 1 << 16;
template <typename W>
__global__ __launch_bounds__(1024) void ln_reduce_kernel(const float* part, int nparts, int c, W* dgamma, W* dbeta) {
  __shared__ float s[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (long first = (long)blockIdx.x * 32; first < 2L * c; first += (long)gridDim.x * 32) {
    const long k = first + tx;
    s[ty][tx] = k < 2L * c ? part_sum(part + k, 2L * c, ty, nparts) : 0.0f;
    __syncthreads();
    if (ty == 0 && k < 2L * c) {
      const float v = pair_sum<32, 33>(&s[0][tx]);
      if (k < c) {
        if (dgamma) dgamma[k] = (W)v;
      } else if (dbeta) {
        dbeta[k - c] = (W)v;
      }
    }
    __syncthreads();
  }
}

// How rows of n vectors are held: by groups of G lanes, or (G = 0) a workgroup of `threads`, I vectors a
// lane; I = 0: too long.  The backward's grid, each workgroup of which writes a partial row, is what a
// compute unit's registers hold at once (16-bit elements 20 waves, f32 32; 4 workgroups of small groups).
struct Group { int G, I, threads, at_once; };
Group group_of(int n, int elem) {
  const int waves = elem == GWN_ELEM_F32 ? 32 : 20;
  for (int g = 4; g <= 64; g *= 2)
    if (n <= g) return {g, 1, THREADS, 4};
  const int w = (n + 63) / 64;
  if (w <= MOST / 64) return {0, 1, w * 64, waves / w > 0 ? waves / w : 1};
  if (w <= MOST / 64 * 2) return {0, 4, MOST / 2, 1};
  return {0, 0, THREADS, 0};
}
int vectors(int c, int elem) { return (int)(((long)c * elem_bytes(elem) + 15) / 16); }

#define LN_GROUPS(X) X(4, 1) X(8, 1) X(16, 1) X(32, 1) X(64, 1) X(0, 1) X(0, 4)

// workgroups of the backward, each with one partial row
int bwd_grid(long rows, int c, int elem) {
  const Group g = group_of(vectors(c, elem), elem);
  if (!g.I) {
    const long by = (rows + 15) / 16;
    return (int)(by < 1 ? 1 : by < 64 ? by : 64);
  }
  const long most = (long)gwn_device_cus() * g.at_once;
  const long per = g.G ? THREADS / g.G : 1, want = (rows + per - 1) / per;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, typename W>
int fwd(const LnFwd& p, int elem, hipStream_t s) {
  const Group g = group_of(vectors(p.c, elem), elem);
  const long per = g.G ? THREADS / g.G : 1, want = (p.rows + per - 1) / per;
  const long most = (long)gwn_device_cus() * (2048 / g.threads);
  const int grid = (int)(want < most ? want : most);
  const bool even = p.c % Vec<T>::N == 0;
#define X(GG, II)                                            \
  if (g.G == GG && g.I == II) {                              \
    (even ? ln_fwd_kernel<T, W, GG, II, true> : ln_fwd_kernel<T, W, GG, II, false>)<<<grid, g.threads, 0, s>>>(p); \
    GWN_CHECK_LAUNCH();                                      \
    return GWN_OK;                                           \
  }
  LN_GROUPS(X)
#undef X
  ln_fwd_long_kernel<T, W><<<grid, THREADS, 0, s>>>(p);
  GWN_CHECK_LAUNCH();
  return GWN_OK;
}

template <typename T, typename W>
int bwd(const LnBwd& p, int elem, void* dgamma, void* dbeta, hipStream_t s) {
  const Group g = group_of(vectors(p.c, elem), elem);
  const int grid = bwd_grid(p.rows, p.c, elem);
  bool done = p.rows == 0;
  const bool even = p.c % Vec<T>::N == 0;
#define X(GG, II)                                            \
  if (!done && g.G == GG && g.I == II) {                     \
    (even ? ln_bwd_kernel<T, W, GG, II, true> : ln_bwd_kernel<T, W, GG, II, false>)<<<grid, g.threads, 0, s>>>(p); \
    GWN_CHECK_LAUNCH();                                      \
    done = true;                                             \
  }
  LN_GROUPS(X)
#undef X
  if (!done) {
    if (p.part) {  // first: dx may overwrite dy
      ln_cols_long_kernel<T><<<dim3((vectors(p.c, elem) + 63) / 64, grid), THREADS, 0, s>>>(p);
      GWN_CHECK_LAUNCH();
    }
    if (p.dx) {
      const long most = (long)gwn_device_cus() * 8;
      ln_bwd_long_kernel<T, W><<<(int)(p.rows < most ? p.rows : most), THREADS, 0, s>>>(p);
      GWN_CHECK_LAUNCH();
    }
  }
  if (!p.part) return GWN_OK;
  const long blocks = (2L * p.c + 31) / 32;
  ln_reduce_kernel<W><<<(int)(blocks < REDUCE_GRID ? blocks : REDUCE_GRID), 1024, 0, s>>>(
      p.part, p.rows ? grid : 0, p.c, (W*)dgamma, (W*)dbeta);
  GWN_CHECK_LAUNCH();
  return GWN_OK;
}

int common_checks(long rows, int c, int elem, long align_bits) {
  GWN_REQUIRE(elem_ok(elem), "layernorm: unknown element type");
  GWN_REQUIRE(rows >= 0 && c > 0, "layernorm: rows must be >= 0 and c > 0");
  GWN_REQUIRE(c <= (1 << 30), "layernorm: c is at most 2^30");
  GWN_REQUIRE((align_bits & (elem_bytes(elem) - 1)) == 0, "layernorm: a pointer is not aligned to its element");
  return GWN_OK;
}

}  // namespace

extern "C" {

int gwn_layernorm_fwd(const void* x, long ldx, long rows, int c, int elem, const void* gamma, const void* beta,
                      int params_f32, float eps, void* y, long ldy, float* mean, float* rstd, hipStream_t stream) {
  const int rc = common_checks(rows, c, elem, (long)x | (long)y);
  if (rc) return rc;
  GWN_REQUIRE(eps >= 0.0f, "layernorm: eps must not be negative");
  GWN_REQUIRE((mean == nullptr) == (rstd == nullptr), "layernorm: mean and rstd come together");
  if (rows == 0) return GWN_OK;
  GWN_REQUIRE(x && y, "layernorm: null pointer");
  GWN_REQUIRE(ldx >= c && ldy >= c, "layernorm: a leading dimension is shorter than the row");
  const long pb = params_f32 ? 3 : elem_bytes(elem) - 1;
  GWN_REQUIRE((((long)gamma | (long)beta) & pb) == 0 && (((long)mean | (long)rstd) & 3) == 0,
              "layernorm: a pointer is not aligned to its element");
  GWN_DEBUG_RANGE(x, ((rows - 1) * ldx + c) * elem_bytes(elem), "layernorm x");
  GWN_DEBUG_RANGE(y, ((rows - 1) * ldy + c) * elem_bytes(elem), "layernorm y");
  const LnFwd p{x, ldx, rows, c, gamma, beta, eps, y, ldy, mean, rstd};
  if (elem == GWN_ELEM_F32) return fwd<float, float>(p, elem, stream);
  if (elem == GWN_ELEM_F16) return params_f32 ? fwd<f16, float>(p, elem, stream) : fwd<f16, f16>(p, elem, stream);
  return params_f32 ? fwd<bf16, float>(p, elem, stream) : fwd<bf16, bf16>(p, elem, stream);
}

long gwn_layernorm_bwd_workspace_floats(long rows, int c, int elem) {
  if (rows < 0 || c <= 0 || !elem_ok(elem)) return 0;
  return (long)bwd_grid(rows, c, elem) * 2 * c;
}

int gwn_layernorm_bwd(const void* dy, long ld_dy, const void* x, long ldx, long rows, int c, int elem,
                      const void* gamma, int params_f32, const float* mean, const float* rstd, void* dx, long ld_dx,
                      void* dgamma, void* dbeta, float* workspace, hipStream_t stream) {
  const int rc = common_checks(rows, c, elem, (long)dy | (long)x | (long)dx);
  if (rc) return rc;
  const bool params = dgamma || dbeta;
  if (!dx && !params) return GWN_OK;
  if (rows == 0 && !params) return GWN_OK;
  GWN_REQUIRE(!params || workspace, "layernorm: the parameters' gradients need a workspace");
  GWN_REQUIRE(rows == 0 || (dy && x && mean && rstd), "layernorm: null pointer");
  GWN_REQUIRE(rows == 0 || (ld_dy >= c && ldx >= c && (!dx || ld_dx >= c)),
              "layernorm: a leading dimension is shorter than the row");
  const long pb = params_f32 ? 3 : elem_bytes(elem) - 1;
  GWN_REQUIRE((((long)gamma | (long)dgamma | (long)dbeta) & pb) == 0 &&
                  (((long)mean | (long)rstd | (long)workspace) & 3) == 0,
              "layernorm: a pointer is not aligned to its element");
  if (rows) {
    GWN_DEBUG_RANGE(dy, ((rows - 1) * ld_dy + c) * elem_bytes(elem), "layernorm dy");
    GWN_DEBUG_RANGE(x, ((rows - 1) * ldx + c) * elem_bytes(elem), "layernorm x");
    GWN_DEBUG_RANGE(dx, ((rows - 1) * ld_dx + c) * elem_bytes(elem), "layernorm dx");
  }
  if (params) GWN_DEBUG_RANGE(workspace, gwn_layernorm_bwd_workspace_floats(rows, c, elem) * 4, "layernorm workspace");
  const LnBwd p{dy, ld_dy, x, ldx, rows, c, gamma, mean, rstd, dx, ld_dx, params ? workspace : nullptr};
  if (elem == GWN_ELEM_F32) return bwd<float, float>(p, elem, dgamma, dbeta, stream);
  if (elem == GWN_ELEM_F16)
    return params_f32 ? bwd<f16, float>(p, elem, dgamma, dbeta, stream)
                      : bwd<f16, f16>(p, elem, dgamma, dbeta, stream);
  return params_f32 ? bwd<bf16, float>(p, elem, dgamma, dbeta, stream)
                    : bwd<bf16, bf16>(p, elem, dgamma, dbeta, stream);
}

}  // extern "C"
