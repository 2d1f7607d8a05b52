// Dropout whose mask is never stored: y_i = r_i + keep(i) x_i / (1 - p), keep(i) from the
// counter-based generator of elem.h; the backward is the same kernel on dy without r.
#include "elem.h"

using namespace elem;

namespace {

// One 16-byte vector per lane and iteration.  Bound by memory: 2 (3 with a residual) transfers per
// element against about 12 VALU operations for its bit of the mask.  85 million elements in bf16: 64 us, with
// a residual 95 us (5.3 TB/s, as a large copy).
template <typename T, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* res, T* y, long count, Drop d) {
  constexpr int V = Vec<T>::N;
  const long step = (long)gridDim.x * 256 * V;
  long i = ((long)blockIdx.x * 256 + threadIdx.x) * V;
  DropKey key;
  key.init(d, i);
  for (; i < count; i += step) {
    key.seek(i);
    if (i + V <= count) {
      const Pack<T, V> a = load<T, V>(x + i);
      Pack<T, V> r, o;
      if (RES) r = load<T, V>(res + i);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float v = key.keep((unsigned)i + j, d.thr) ? (float)a.v[j] * d.scale : 0.0f;
        o.v[j] = (T)(RES ? v + (float)r.v[j] : v);
      }
      store<T, V>(y + i, o);
    } else {
      for (int j = 0; i + j < count; ++j) {
        const float v = key.keep((unsigned)i + j, d.thr) ? (float)x[i + j] * d.scale : 0.0f;
        y[i + j] = (T)(RES ? v + (float)res[i + j] : v);
      }
    }
  }
}

template <typename T>
int run(const void* x, const void* res, void* y, long count, const Drop& d, hipStream_t s) {
  const long vecs = (count + Vec<T>::N - 1) / Vec<T>::N;
  const long want = (vecs + 255) / 256, most = (long)gwn_device_cus() * 32;
  const int grid = (int)(want < most ? want : most);
  if (res)
    dropout_kernel<T, true><<<grid, 256, 0, s>>>((const T*)x, (const T*)res, (T*)y, count, d);
  else
    dropout_kernel<T, false><<<grid, 256, 0, s>>>((const T*)x, nullptr, (T*)y, count, d);
  GWN_CHECK_LAUNCH();
  return GWN_OK;
}

}  // namespace

extern "C" int gwn_dropout(const void* x, const void* residual, void* y, long count, int elem,
                           const unsigned long long* seed_ptr, unsigned long long salt, double drop_p,
                           hipStream_t stream) {
  GWN_REQUIRE(elem_ok(elem), "dropout: unknown element type");
  GWN_REQUIRE(count >= 0, "dropout: negative count");
  GWN_REQUIRE(drop_p >= 0.0 && drop_p <= 1.0, "dropout: the rate must be between 0 and 1");
  if (count == 0) return GWN_OK;
  GWN_REQUIRE(x && y && seed_ptr, "dropout: null pointer");
  const long align = elem_bytes(elem) - 1;
  GWN_REQUIRE((((size_t)x | (size_t)y | (size_t)residual) & align) == 0 && ((size_t)seed_ptr & 7) == 0,
              "dropout: a pointer is not aligned to its element");
  GWN_DEBUG_RANGE(x, count * elem_bytes(elem), "dropout x");
  GWN_DEBUG_RANGE(residual, count * elem_bytes(elem), "dropout residual");
  GWN_DEBUG_RANGE(y, count * elem_bytes(elem), "dropout y");
  const Drop d = drop_of(seed_ptr, salt, drop_p);
  if (elem == GWN_ELEM_F32) return run<float>(x, residual, y, count, d, stream);
  if (elem == GWN_ELEM_F16) return run<f16>(x, residual, y, count, d, stream);
  return run<bf16>(x, residual, y, count, d, stream);
}
