// y = residual + D(act(x w^T + bias)) in one launch, and its gradients.
//
//   z = x w^T + b,  y = r + D(act(z));  dz = D'(dy) act'(z),  db = sum_m dz,  dx = dz w,  dw = dz^T x
#include "elem.h"

using namespace elem;

namespace {

// the saved pre-activation: float beside f32 elements, else f16
template <typename T> struct ZType { typedef f16 type; };
template <> struct ZType<float> { typedef float type; };

__device__ __forceinline__ void put_z(float* p, float z) { *p = z; }
__device__ __forceinline__ void put_z(f16* p, float z) {
  // finite values stay finite, and a positive one positive: the derivatives' limits and relu's
  // border then come out of the rounded value as out of the exact one
  f16 h = (f16)(fabsf(z) < 3.0e38f ? fminf(fmaxf(z, -65504.0f), 65504.0f) : z);
  if (z > 0.0f && h == (f16)0.0f) h = (f16)5.9604645e-8f;
  *p = h;
}

struct Epi {
  const void* bias;
  const void* res; long ld_res;
  void* z; long ldz;
  int act;
  Drop drop;
};

// C(m, n) = epi(sum_k A[m sam + k sak] B[n sbn + k sbk]), C [M][ldc]
struct Gemm {
  const void* A; long sam, sak;
  const void* B; long sbn, sbk;
  void* C; long ldc;
  int M, N, K;
  Epi e;
};

template <typename T>
__device__ __forceinline__ void epilogue(const Gemm& p, DropKey& key, long m, long n, float v) {
  if (p.e.bias) v += (float)((const T*)p.e.bias)[n];
  if (p.e.z) put_z((typename ZType<T>::type*)p.e.z + m * p.e.ldz + n, v);
  v = act_value<is16<T>>(v, p.e.act);
  if (p.e.drop.thr) {
    const unsigned long long i = (unsigned long long)m * p.N + n;
    key.seek(i);
    v = key.keep((unsigned)i, p.e.drop.thr) ? v * p.e.drop.scale : 0.0f;
  }
  if (p.e.res) v += (float)((const T*)p.e.res)[m * p.e.ld_res + n];
  ((T*)p.C)[m * p.ldc + n] = (T)v;
}

template <typename T>
__global__ __launch_bounds__(256) void gemm_kernel(const Gemm p) {
  __shared__ float As[16][65], Bs[16][65];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long m0 = (long)blockIdx.x * 64, n0 = (long)blockIdx.y * 64;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 16) {
    for (int q = threadIdx.x; q < 1024; q += 256) {
      const int i = p.sak == 1 ? q >> 4 : q & 63, k = p.sak == 1 ? q & 15 : q >> 6;
      As[k][i] = m0 + i < p.M && k0 + k < p.K ? (float)((const T*)p.A)[(m0 + i) * p.sam + (long)(k0 + k) * p.sak] : 0.0f;
    }
    for (int q = threadIdx.x; q < 1024; q += 256) {
      const int i = p.sbk == 1 ? q >> 4 : q & 63, k = p.sbk == 1 ? q & 15 : q >> 6;
      Bs[k][i] = n0 + i < p.N && k0 + k < p.K ? (float)((const T*)p.B)[(n0 + i) * p.sbn + (long)(k0 + k) * p.sbk] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += As[k][ty * 4 + i] * Bs[k][tx + 16 * j];
    __syncthreads();
  }
  DropKey key;
  if (p.e.drop.thr) key.init(p.e.drop, (unsigned long long)m0 * p.N + n0);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
      if (m < p.M && n < p.N) epilogue<T>(p, key, m, n, acc[i][j]);
    }
}

template <typename T>
int gemm(const Gemm& p, hipStream_t s) {
  gemm_kernel<T><<<dim3((p.M + 63) / 64, (p.N + 63) / 64), 256, 0, s>>>(p);
  GWN_CHECK_LAUNCH();
  return GWN_OK;
}

struct Dz {
  const void* dy; long ld_dy;
  const void* z; long ldz;
  void* dz;     // [M][N], NULL = not written (dz is dy)
  float* part;  // [gridDim.y][N] column sums, NULL = not wanted
  int M, N, act;
  Drop drop;
};

// 256 columns x a stripe of rows a workgroup
template <typename T>
__global__ __launch_bounds__(256) void dz_kernel(const Dz p) {
  const long n = (long)blockIdx.x * 256 + threadIdx.x;
  if (n >= p.N) return;
  DropKey key;
  if (p.drop.thr) key.init(p.drop, (unsigned long long)blockIdx.y * p.N);
  float sum = 0.0f;
  for (long m = blockIdx.y; m < p.M; m += gridDim.y) {
    float v = (float)((const T*)p.dy)[m * p.ld_dy + n];
    if (p.drop.thr) {
      const unsigned long long i = (unsigned long long)m * p.N + n;
      key.seek(i);
      v = key.keep((unsigned)i, p.drop.thr) ? v * p.drop.scale : 0.0f;
    }
    if (p.act != GWN_ACT_NONE)
      v *= act_slope<is16<T>>((float)((const typename ZType<T>::type*)p.z)[m * p.ldz + n], p.act);
    sum += v;
    if (p.dz) ((T*)p.dz)[m * p.N + n] = (T)v;
  }
  if (p.part) p.part[(long)blockIdx.y * p.N + n] = sum;
}

template <typename T>
__global__ __launch_bounds__(256) void colsum_kernel(const float* part, int nparts, int n, T* out) {
  const long k = (long)blockIdx.x * 256 + threadIdx.x;
  if (k >= n) return;
  float v = 0.0f;
  for (int q = 0; q < nparts; ++q) v += part[(long)q * n + k];
  out[k] = (T)v;
}

int dz_parts(int M) { return M < 1 ? 1 : M < 256 ? M : 256; }

template <typename T>
int fwd(const gwn_linear_args* a, hipStream_t s) {
  Gemm p{a->x, a->ldx, 1, a->w, a->ldw, 1, a->y, a->ldy, a->M, a->N, a->K, {}};
  p.e = {a->bias, a->residual, a->ld_res, a->act == GWN_ACT_NONE ? nullptr : a->z, a->ldz, a->act,
         drop_of(a->seed_ptr, a->salt, a->drop_p)};
  return gemm<T>(p, s);
}

template <typename T>
int bwd(const gwn_linear_bwd_args* a, hipStream_t s) {
  const Drop drop = drop_of(a->seed_ptr, a->salt, a->drop_p);
  const bool changes = a->act != GWN_ACT_NONE || drop.thr;
  const bool product = a->dx || a->dw;
  const int parts = dz_parts(a->M);
  T* dzbuf = (T*)(a->workspace + (long)parts * a->N);
  const T* dz = changes ? dzbuf : (const T*)a->dy;
  const long ld = changes ? a->N : a->ld_dy;
  if ((changes && product) || a->dbias) {
    const Dz q{a->dy, a->ld_dy, a->z, a->ldz, changes && product ? dzbuf : nullptr, a->dbias ? a->workspace : nullptr,
               a->M, a->N, a->act, drop};
    dz_kernel<T><<<dim3((a->N + 255) / 256, parts), 256, 0, s>>>(q);
    GWN_CHECK_LAUNCH();
  }
  if (a->dbias) {
    colsum_kernel<T><<<(a->N + 255) / 256, 256, 0, s>>>(a->workspace, parts, a->N, (T*)a->dbias);
    GWN_CHECK_LAUNCH();
  }
  if (a->dx && a->M) {
    Gemm p{dz, ld, 1, a->w, 1, a->ldw, a->dx, a->ld_dx, a->M, a->K, a->N, {}};
    const int rc = gemm<T>(p, s);
    if (rc) return rc;
  }
  if (a->dw) {
    Gemm p{dz, 1, ld, a->x, 1, a->ldx, a->dw, a->ld_dw, a->N, a->K, a->M, {}};
    const int rc = gemm<T>(p, s);
    if (rc) return rc;
  }
  return GWN_OK;
}

long range_bytes(long rows, long ld, long cols, int bytes) { return rows ? ((rows - 1) * ld + cols) * bytes : 0; }

int shape_checks(int M, int N, int K, int elem, int act, double drop_p, const void* seed_ptr) {
  GWN_REQUIRE(elem_ok(elem), "linear: unknown element type");
  GWN_REQUIRE(act >= GWN_ACT_NONE && act <= GWN_ACT_SILU, "linear: unknown activation");
  GWN_REQUIRE(M >= 0 && N > 0 && K > 0, "linear: M must be >= 0, N and K > 0");
  GWN_REQUIRE(M <= (1 << 30) && N <= (1 << 21) && K <= (1 << 21), "linear: M is at most 2^30, N and K 2^21");
  GWN_REQUIRE(drop_p >= 0.0 && drop_p <= 1.0, "linear: the dropout rate must be between 0 and 1");
  GWN_REQUIRE(drop_p == 0.0 || (seed_ptr && ((size_t)seed_ptr & 7) == 0), "linear: dropout needs a seed");
  return GWN_OK;
}

}  // namespace

extern "C" {

long gwn_linear_fwd_workspace_floats(int M, int N, int K, int elem) {
  (void)M, (void)N, (void)K, (void)elem;
  return 0;
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
  const long ws = gwn_linear_fwd_workspace_floats(a->M, a->N, a->K, a->elem);
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

long gwn_linear_bwd_workspace_floats(int M, int N, int K, int elem) {
  if (M < 0 || N <= 0 || K <= 0 || !elem_ok(elem)) return 0;
  return (long)dz_parts(M) * N + ((long)M * N * elem_bytes(elem) + 3) / 4;
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
  GWN_REQUIRE(a->workspace && ((size_t)a->workspace & 15) == 0, "linear_bwd: the workspace is missing");
  GWN_DEBUG_RANGE(a->dy, range_bytes(a->M, a->ld_dy, a->N, e), "linear_bwd dy");
  if (a->dw) GWN_DEBUG_RANGE(a->x, range_bytes(a->M, a->ldx, a->K, e), "linear_bwd x");
  if (a->dx) GWN_DEBUG_RANGE(a->w, range_bytes(a->N, a->ldw, a->K, e), "linear_bwd w");
  if (a->act != GWN_ACT_NONE)
    GWN_DEBUG_RANGE(a->z, range_bytes(a->M, a->ldz, a->N, a->elem == GWN_ELEM_F32 ? 4 : 2), "linear_bwd z");
  GWN_DEBUG_RANGE(a->dx, range_bytes(a->M, a->ld_dx, a->K, e), "linear_bwd dx");
  GWN_DEBUG_RANGE(a->dw, range_bytes(a->N, a->ld_dw, a->K, e), "linear_bwd dw");
  GWN_DEBUG_RANGE(a->workspace, gwn_linear_bwd_workspace_floats(a->M, a->N, a->K, a->elem) * 4, "linear_bwd workspace");
  if (a->elem == GWN_ELEM_F32) return bwd<float>(a, stream);
  if (a->elem == GWN_ELEM_F16) return bwd<f16>(a, stream);
  return bwd<bf16>(a, stream);
}

}  // extern "C"
