// Distillation from a teacher's top logits.  A row has V student logits z and K teacher logits t_k
// at the vocabulary ids i_k (an id below 0 or beyond V: no entry).  With a temperature tau,
//
//   p = softmax over the entries of t/tau,   q = softmax(z/tau) over the whole vocabulary
//   loss = tau^2 * sum_k p_k (log p_k - log q_{i_k})
//   dz_v = g * tau * (q_v - sum_{k: i_k = v} p_k)
//
// A row without entries has loss 0 and gradient 0.  The forward reads the logits once (running
// maximum and sum) and keeps log(sum exp(z/tau)); the backward reads them once more and writes dz.
#include "lsh_lm.h"

namespace lsh {

constexpr int kDsThreads = 256;

// (maximum, sum of exp(x - maximum)) of two parts
__device__ __forceinline__ void lse_join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float a = m == top ? 1.0f : expf(m - top), b = m2 == top ? 1.0f : expf(m2 - top);
  s = s * a + s2 * b;
  m = top;
}

// Element i of an array of either type
template <class T>
__device__ __forceinline__ float ds_value(const void* p, int64_t i, bool f32) {
  return f32 ? ((const float*)p)[i] : to_f(((const T*)p)[i]);
}

// The teacher's distribution of a row, in LDS: p[k] and id[k] (-1: no entry).  Returns whether the
// row has an entry of weight.
template <class T>
__device__ __forceinline__ bool ds_teacher(const void* t, bool t_f32, const int64_t* ids, int64_t row,
                                           int K, int64_t V, float itau, float* p, int* id, float* red) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    float m = -INFINITY;
    for (int k = lane; k < K; k += 64) {
      const int64_t i = ids[row * K + k];
      const bool there = i >= 0 && i < V;
      id[k] = there ? (int)i : -1;
      p[k] = there ? ds_value<T>(t, row * K + k, t_f32) * itau : -INFINITY;
      m = fmaxf(m, p[k]);
    }
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    float s = 0.0f;
    for (int k = lane; k < K; k += 64) {
      p[k] = m > -INFINITY ? expf(p[k] - m) : 0.0f;
      s += p[k];
    }
    s = wave_sum_f(s);
    for (int k = lane; k < K; k += 64) p[k] = s != 0.0f ? p[k] / s : 0.0f;
    if (lane == 0) red[0] = s;
  }
  __syncthreads();
  return red[0] != 0.0f;
}

template <class T>
__global__ __launch_bounds__(kDsThreads) void k_distill(const T* __restrict__ z, int64_t stride,
                                                        const void* __restrict__ tv, bool tv_f32,
                                                        const int64_t* __restrict__ ti,
                                                        float* __restrict__ loss, float* __restrict__ lse,
                                                        int64_t V, int K, float tau) {
  extern __shared__ float s_dyn[];
  float* p = s_dyn;
  int* id = (int*)(s_dyn + K);
  __shared__ float s_m[kDsThreads / 64], s_s[kDsThreads / 64], red[1];
  const int64_t row = blockIdx.x;
  z += row * stride;
  const float itau = 1.0f / tau;
  const bool some = ds_teacher<T>(tv, tv_f32, ti, row, K, V, itau, p, id, red);
  float m = -INFINITY, s = 0.0f;
  for (int64_t v = threadIdx.x; v < V; v += kDsThreads) lse_join(m, s, to_f(z[v]) * itau, 1.0f);
  for (int o = 32; o > 0; o >>= 1) lse_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
  if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = m, s_s[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x < 64) {
    m = s_m[0], s = s_s[0];
    for (int w = 1; w < kDsThreads / 64; ++w) lse_join(m, s, s_m[w], s_s[w]);
    const float l = m + logf(s);
    float sum = 0.0f;
    for (int k = threadIdx.x; k < K; k += 64)
      if (id[k] >= 0 && p[k] > 0.0f) sum += p[k] * (logf(p[k]) - (to_f(z[id[k]]) * itau - l));
    sum = wave_sum_f(sum);
    if (threadIdx.x == 0) {
      loss[row] = some ? tau * tau * sum : 0.0f;
      lse[row] = l;
    }
  }
}

template <class T>
__global__ __launch_bounds__(kDsThreads) void k_distill_bwd(const T* __restrict__ z, int64_t stride,
                                                            const void* __restrict__ tv, bool tv_f32,
                                                            const int64_t* __restrict__ ti,
                                                            const float* __restrict__ lse,
                                                            const float* __restrict__ g, int64_t g_stride,
                                                            T* __restrict__ dz, int64_t V, int K, float tau) {
  extern __shared__ float s_dyn[];
  float* p = s_dyn;
  int* id = (int*)(s_dyn + K);
  __shared__ float red[1];
  const int64_t row = blockIdx.x;
  z += row * stride;
  dz += row * V;
  const float itau = 1.0f / tau, l = lse[row];
  const bool some = ds_teacher<T>(tv, tv_f32, ti, row, K, V, itau, p, id, red);
  const float f = g[row * g_stride] * tau;
  for (int64_t v = threadIdx.x; v < V; v += kDsThreads)
    dz[v] = from_f<T>(some ? f * expf(to_f(z[v]) * itau - l) : 0.0f);
  __syncthreads();  // the rows' entries are written again with the teacher's part
  if (!some) return;
  for (int k = threadIdx.x; k < K; k += kDsThreads) {
    const int v = id[k];
    bool first = v >= 0;
    float sum = 0.0f;
    for (int j = 0; j < K && first; ++j)
      if (id[j] == v) {
        first = j >= k;
        sum += p[j];
      }
    if (first) dz[v] = from_f<T>(f * (expf(to_f(z[v]) * itau - l) - sum));
  }
}

static int ds_check(int dtype, int v_dtype, int64_t rows, int64_t V, int K, float tau) {
  if (!lm_dtype_ok(dtype) || (v_dtype != LSH_F32 && v_dtype != dtype) || !(tau > 0.0f) || !(tau < INFINITY)) return LSH_ERR_ARG;
  if (rows < 0 || rows > 0x7fffffff || V < 1 || V > 0x7fffffff || K < 0 || K > LSH_DISTILL_MAX_K)
    return LSH_ERR_SHAPE;
  return LSH_OK;
}

}  // namespace lsh

using namespace lsh;

extern "C" int lsh_distill_fwd(int dtype, const void* logits, int64_t stride, int v_dtype, const void* values,
                               const int64_t* index, float* loss, float* lse, int64_t rows, int64_t V,
                               int K, float tau, void* stream) {
  if (int rc = ds_check(dtype, v_dtype, rows, V, K, tau)) return rc;
  if (rows == 0) return LSH_OK;
  if (bad_ptr(logits) || (K > 0 && (bad_ptr(values) || bad_ptr(index))) || bad_ptr(loss) || bad_ptr(lse))
    return LSH_ERR_ARG;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_distill<T><<<dim3((unsigned)rows), kDsThreads, (size_t)K * 8, (hipStream_t)stream>>>(
        (const T*)logits, stride, values, v_dtype == LSH_F32, index, loss, lse, V, K, tau);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" int lsh_distill_bwd(int dtype, const void* logits, int64_t stride, int v_dtype, const void* values,
                               const int64_t* index, const float* lse, const float* g, int64_t g_stride,
                               void* dlogits, int64_t rows, int64_t V, int K, float tau, void* stream) {
  if (int rc = ds_check(dtype, v_dtype, rows, V, K, tau)) return rc;
  if (rows == 0) return LSH_OK;
  if (bad_ptr(logits) || (K > 0 && (bad_ptr(values) || bad_ptr(index))) || bad_ptr(lse) || bad_ptr(g) ||
      bad_ptr(dlogits))
    return LSH_ERR_ARG;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_distill_bwd<T><<<dim3((unsigned)rows), kDsThreads, (size_t)K * 8, (hipStream_t)stream>>>(
        (const T*)logits, stride, values, v_dtype == LSH_F32, index, lse, g, g_stride, (T*)dlogits, V, K, tau);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
