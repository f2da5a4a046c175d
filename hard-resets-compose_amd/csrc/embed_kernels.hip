// Embedding lookup with scaling, and the table's gradient.
//
//   out[i] = scale * W[tok_i]          dW[v] = scale * sum_{i: tok_i = v} dout[i]
//
// Ids outside the table and the padding id read as zero rows and leave no gradient.  The gradient
// sums the rows of a token in the order of their positions, in fp32, with no atomics: the same bits
// on every run.
#include "lsh_lm.h"

namespace lsh {

template <class T>
__global__ __launch_bounds__(256) void k_embed(const int64_t* __restrict__ tok, const T* __restrict__ W,
                                               T* __restrict__ out, int64_t V, int D, int64_t pad,
                                               float scale) {
  const int64_t i = blockIdx.x, v = tok[i];
  const bool there = v >= 0 && v < V && v != pad;
  for (int d = threadIdx.x; d < D; d += 256)
    out[(size_t)i * D + d] = there ? from_f<T>(scale * to_f(W[(size_t)v * D + d])) : from_f<T>(0.0f);
}

template <class T>
__global__ __launch_bounds__(256) void k_embed_bwd(const int64_t* __restrict__ tok,
                                                   const T* __restrict__ dout, T* __restrict__ dW,
                                                   int64_t n, int64_t V, int D, int64_t pad, float scale) {
  const int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (v >= V) return;
  for (int d0 = 0; d0 < D; d0 += 64) {
    const int d = d0 + lane;
    float s = 0.0f;
    if (v != pad) {
      for (int64_t i0 = 0; i0 < n; i0 += 64) {
        unsigned long long hit = wave_ballot(i0 + lane < n && tok[i0 + lane] == v);
        while (hit) {
          const int64_t i = i0 + __builtin_ctzll(hit);
          hit &= hit - 1;
          if (d < D) s += to_f(dout[(size_t)i * D + d]);
        }
      }
    }
    if (d < D) dW[(size_t)v * D + d] = from_f<T>(scale * s);
  }
}

static int embed_check(int dtype, int64_t n, int64_t V, int64_t D) {
  if (!lm_dtype_ok(dtype)) return LSH_ERR_ARG;
  if (n < 0 || n > 0x7fffffff || V < 0 || V > 0x7fffffff || D < 1 || D > 0x7fffffff / 4) return LSH_ERR_SHAPE;
  return LSH_OK;
}

}  // namespace lsh

using namespace lsh;

extern "C" int lsh_embed_fwd(int dtype, const int64_t* tokens, const void* weight, void* out, int64_t n,
                             int64_t V, int64_t D, int64_t padding, float scale, void* stream) {
  if (int rc = embed_check(dtype, n, V, D)) return rc;
  if (n == 0) return LSH_OK;
  if (bad_ptr(tokens) || (V > 0 && bad_ptr(weight)) || bad_ptr(out)) return LSH_ERR_ARG;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_embed<T><<<dim3((unsigned)n), 256, 0, (hipStream_t)stream>>>(tokens, (const T*)weight, (T*)out, V,
                                                                  (int)D, padding, scale);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" int lsh_embed_bwd(int dtype, const int64_t* tokens, const void* dout, void* dweight, int64_t n,
                             int64_t V, int64_t D, int64_t padding, float scale, void* stream) {
  if (int rc = embed_check(dtype, n, V, D)) return rc;
  if (V == 0) return LSH_OK;
  if (bad_ptr(dweight) || (n > 0 && (bad_ptr(tokens) || bad_ptr(dout)))) return LSH_ERR_ARG;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_embed_bwd<T><<<dim3((unsigned)((V + 3) / 4)), 256, 0, (hipStream_t)stream>>>(
        tokens, (const T*)dout, (T*)dweight, n, V, (int)D, padding, scale);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
