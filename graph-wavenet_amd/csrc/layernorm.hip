// Layer norm over the last axis, forward and backward.
//
//   mean = sum x / C,  rstd = (sum (x - mean)^2 / C + eps)^(-1/2),  y = (x - mean) rstd g + b
//   xh = (x - mean) rstd,  h = dy g,  dx = rstd (h - sum(h) / C - xh sum(h xh) / C)
//   dg = sum_rows dy xh,  db = sum_rows dy
//
// Bound by memory: x read and y written once forward; x and dy read, dx written once backward.  A
// row lives in the registers of a group of G lanes (G = 4 .. 64 lanes of a wave, or a whole
// workgroup), I 16-byte vectors a lane, so that the variance is the centred sum of squares and
// nothing is read twice.  The centred values' own mean is taken off again (the corrected two-pass
// form): the first mean's rounding, which 1 / sqrt(eps) would magnify in a row that hardly varies,
// drops out, and a constant row gives exactly b.  Groups walk the rows; each lane keeps its columns' sums of dg and db in
// registers over all rows its group sees, a workgroup adds its groups up and writes one partial row,
// and a second launch adds the partial rows in a fixed order.  Rows longer than a workgroup's
// registers are looped over (they stay in the L2 cache between the passes).
#include "elem.h"

using namespace elem;

namespace {

constexpr int THREADS = 256;

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

// sum over the G lanes of a group, the same value in all of them
template <int G>
__device__ __forceinline__ float group_sum(float v, float* lds) {
#pragma unroll
  for (int o = 1; o < (G < 64 ? G : 64); o <<= 1) v += __shfl_xor(v, o, 64);
  if (G > 64) {
    __syncthreads();  // the last sum's reads are done
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v += lds[w];
  }
  return v;
}

template <typename T, typename W, int G, int I>
__global__ __launch_bounds__(THREADS) void ln_fwd_kernel(const LnFwd p) {
  constexpr int V = Vec<T>::N;
  __shared__ float red[THREADS / 64];
  const int lane = threadIdx.x % G;
  const float c = (float)p.c;
  constexpr int PER = THREADS / G;
  const long step = (long)gridDim.x * PER;
  // whole groups leave together; a whole workgroup where the group is one
  for (long row = (long)blockIdx.x * PER + threadIdx.x / G; row < p.rows; row += step) {
    const T* x = (const T*)p.x + row * p.ldx;
    float v[I][V], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int at = (lane + G * i) * V;
      load_f<T, V>(v[i], x + at, p.c - at, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) sum += v[i][j];
    float mean = group_sum<G>(sum, red) / c, sq = 0.0f, sd = 0.0f;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int rem = p.c - (lane + G * i) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = j < rem ? v[i][j] - mean : 0.0f;
        sq += v[i][j] * v[i][j];
        sd += v[i][j];
      }
    }
    const float left = group_sum<G>(sd, red) / c;
    const float rstd = 1.0f / sqrtf(fmaxf(group_sum<G>(sq, red) / c - left * left, 0.0f) + p.eps);
    mean += left;
    if (p.mean && lane == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
    T* y = (T*)p.y + row * p.ldy;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int at = (lane + G * i) * V, rem = p.c - at;
      if (rem > 0) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = (v[i][j] - left) * rstd;
        if (p.gamma) {
          float g[V];
          load_f<W, V>(g, (const W*)p.gamma + at, rem, 0.0f);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] *= g[j];
        }
        if (p.beta) {
          float b[V];
          load_f<W, V>(b, (const W*)p.beta + at, rem, 0.0f);
#pragma unroll
          for (int j = 0; j < V; ++j) o[j] += b[j];
        }
        store_f<T, V>(y + at, o, rem);
      }
    }
  }
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
    const float first = group_sum<THREADS>(sum, red) / c;
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
    const float left = group_sum<THREADS>(sd, red) / c, mean = first + left;
    const float rstd = 1.0f / sqrtf(fmaxf(group_sum<THREADS>(sq, red) / c - left * left, 0.0f) + p.eps);
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

template <typename T, typename W, int G, int I>
__global__ __launch_bounds__(THREADS) void ln_bwd_kernel(const LnBwd p) {
  constexpr int V = Vec<T>::N, PER = THREADS / G;
  __shared__ float red[THREADS / 64];
  __shared__ float cols[PER > 1 ? 2 * G * I * V : 1];
  const int lane = threadIdx.x % G;
  const float inv = 1.0f / (float)p.c;
  float dg[I][V] = {}, db[I][V] = {};
  const long step = (long)gridDim.x * PER;
  for (long row = (long)blockIdx.x * PER + threadIdx.x / G; row < p.rows; row += step) {
    const T* x = (const T*)p.x + row * p.ldx;
    const T* dy = (const T*)p.dy + row * p.ld_dy;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float v[I][V], h[I][V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int at = (lane + G * i) * V, rem = p.c - at;
      load_f<T, V>(v[i], x + at, rem, mean);
      load_f<T, V>(h[i], dy + at, rem, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int at = (lane + G * i) * V, rem = p.c - at;
      float g[V];
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = 1.0f;
      if (p.gamma && rem > 0) load_f<W, V>(g, (const W*)p.gamma + at, rem, 0.0f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = (v[i][j] - mean) * rstd;
        dg[i][j] += h[i][j] * v[i][j];
        db[i][j] += h[i][j];
        h[i][j] *= g[j];
        s1 += h[i][j];
        s2 += h[i][j] * v[i][j];
      }
    }
    if (!p.dx) continue;
    s1 = group_sum<G>(s1, red) * inv;
    s2 = group_sum<G>(s2, red) * inv;
    T* dx = (T*)p.dx + row * p.ld_dx;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int at = (lane + G * i) * V, rem = p.c - at;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = rstd * (h[i][j] - s1 - v[i][j] * s2);
      if (rem > 0) store_f<T, V>(dx + at, o, rem);
    }
  }
  if (!p.part) return;
  float* part = p.part + (long)blockIdx.x * 2 * p.c;
  if constexpr (PER == 1) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int at = (lane + G * i) * V, rem = p.c - at;
      if (rem > 0) {
        store_f<float, V>(part + at, dg[i], rem);
        store_f<float, V>(part + p.c + at, db[i], rem);
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
          for (int j = 0; j < V; ++j) {
            const int at = (lane + G * i) * V + j;
            cols[at] = w ? cols[at] + dg[i][j] : dg[i][j];
            cols[G * I * V + at] = w ? cols[G * I * V + at] + db[i][j] : db[i][j];
          }
      }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < p.c; k += THREADS) {
      part[k] = cols[k];
      part[p.c + k] = cols[G * I * V + k];
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
        s1 = group_sum<THREADS>(s1, red) * inv;
        s2 = group_sum<THREADS>(s2, red) * inv;
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

// out[k] = sum over parts of part[.][k]: 32 columns x 32 lanes of parts a workgroup, fixed order
template <typename W>
__global__ __launch_bounds__(1024) void ln_reduce_kernel(const float* part, int nparts, int c, W* dgamma, W* dbeta) {
  __shared__ float s[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long k = (long)blockIdx.x * 32 + tx;
  float v = 0.0f;
  if (k < 2L * c)
#pragma unroll 8
    for (int q = ty; q < nparts; q += 32) v += part[(long)q * 2 * c + k];
  s[ty][tx] = v;
  __syncthreads();
  if (ty == 0 && k < 2L * c) {
    v = 0.0f;
#pragma unroll
    for (int q = 0; q < 32; ++q) v += s[q][tx];
    if (k < c) {
      if (dgamma) dgamma[k] = (W)v;
    } else if (dbeta) {
      dbeta[k - c] = (W)v;
    }
  }
}

// the group that holds a row of n vectors: lanes G and vectors a lane I; G = 0: too long
struct Group { int G, I; };
Group group_of(int n) {
  if (n <= 4) return {4, 1};
  if (n <= 8) return {8, 1};
  if (n <= 16) return {16, 1};
  if (n <= 32) return {32, 1};
  if (n <= 256) return {64, (n + 63) / 64};
  const int i = (n + 255) / 256;
  if (i <= 4) return {256, i};
  if (i <= 6) return {256, 6};
  if (i <= 8) return {256, 8};
  return {0, 0};
}
int vectors(int c, int elem) { return (int)(((long)c * elem_bytes(elem) + 15) / 16); }

#define LN_GROUPS(X) \
  X(4, 1) X(8, 1) X(16, 1) X(32, 1) X(64, 1) X(64, 2) X(64, 3) X(64, 4) X(256, 2) X(256, 3) X(256, 4) X(256, 6) X(256, 8)

// workgroups of the backward, each with one partial row
int bwd_grid(long rows, int c, int elem) {
  const Group g = group_of(vectors(c, elem));
  const long most = (long)gwn_device_cus() * 2;
  if (!g.G) {
    const long by = (rows + 15) / 16;
    return (int)(by < 1 ? 1 : by < 64 ? by : 64);
  }
  const long per = THREADS / g.G, want = (rows + per - 1) / per;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, typename W>
int fwd(const LnFwd& p, int elem, hipStream_t s) {
  const Group g = group_of(vectors(p.c, elem));
  const long per = g.G ? THREADS / g.G : 1, want = (p.rows + per - 1) / per, most = (long)gwn_device_cus() * 16;
  const int grid = (int)(want < most ? want : most);
#define X(GG, II)                                            \
  if (g.G == GG && g.I == II) {                              \
    ln_fwd_kernel<T, W, GG, II><<<grid, THREADS, 0, s>>>(p); \
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
  const Group g = group_of(vectors(p.c, elem));
  const int grid = bwd_grid(p.rows, p.c, elem);
  bool done = p.rows == 0;
#define X(GG, II)                                            \
  if (!done && g.G == GG && g.I == II) {                     \
    ln_bwd_kernel<T, W, GG, II><<<grid, THREADS, 0, s>>>(p); \
    GWN_CHECK_LAUNCH();                                      \
    done = true;                                             \
  }
  LN_GROUPS(X)
#undef X
  if (!done) {
    if (p.dx) {
      const long most = (long)gwn_device_cus() * 8;
      ln_bwd_long_kernel<T, W><<<(int)(p.rows < most ? p.rows : most), THREADS, 0, s>>>(p);
      GWN_CHECK_LAUNCH();
    }
    if (p.part) {
      ln_cols_long_kernel<T><<<dim3((vectors(p.c, elem) + 63) / 64, grid), THREADS, 0, s>>>(p);
      GWN_CHECK_LAUNCH();
    }
  }
  if (!p.part) return GWN_OK;
  ln_reduce_kernel<W><<<(int)((2L * p.c + 31) / 32), 1024, 0, s>>>(p.part, p.rows ? grid : 0, p.c, (W*)dgamma,
                                                                   (W*)dbeta);
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
