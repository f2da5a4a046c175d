// Distillation from a teacher's top logits.  A row has V student logits z and K teacher logits t_k
// at the vocabulary ids i_k (an id below 0 or beyond V: no entry).  With a temperature tau,
//
//   p = softmax over the entries of t/tau,   q = softmax(z/tau) over the whole vocabulary
//   loss = tau^2 * sum_k p_k (log p_k - log q_{i_k})
//   dz_v = g * tau * (q_v - sum_{k: i_k = v} p_k)
//
// A row without entries has loss 0 and gradient 0.  All exponents are in base 2: with c = log2(e)/tau,
// m the largest logit and l = log2(sum 2^(c*(z - m))), q_v = 2^(c*(z_v - m) - l).  (m stays apart from l:
// their sum would round by a share of the logits' size where only their differences matter.)  The
// forward reads the logits once, with the running maximum and sum of the softmax, and keeps m, l and the
// teacher's two; the backward reads them once more and writes dz.  Both are bound by the logits' bytes:
// 4096 x 32000 bf16 with 64 entries, one after the other in training, 81 us forward (262 MB; 53 where no gradient of
// before is still on its way to memory) and 92 backward (524 MB): 4.5 TB/s over both.  A row is split over several
// workgroups where there are too few rows for the chip, and the parts' maxima and sums are joined in order.
#include <algorithm>

#include "lsh_lm.h"

namespace lsh {

constexpr int kDsThreads = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DsArgs {
  const void* z;
  int64_t stride;
  const void* t;
  bool t_f32;
  const int64_t* id;
  float* loss;
  float* stats;  // [4, rows]: m and l, and the teacher's (-inf: no entry)
  float* part;   // [rows, splits, 2]: maximum and sum of each part
  const float* g;
  int64_t g_stride;
  void* dz;
  int64_t rows, V;
  int K, splits;
  int64_t len;  // logits of a part
  float c, tau;
};

// (maximum, sum of 2^(c*(x - maximum))) of two parts; a part without values has maximum -inf, sum 0
__device__ __forceinline__ void ds_join(float& m, float& s, float m2, float s2, float c) {
  const float top = fmaxf(m, m2), at = top > -INFINITY ? top : 0.0f;
  s = s * __builtin_amdgcn_exp2f((m - at) * c) + s2 * __builtin_amdgcn_exp2f((m2 - at) * c);
  m = top;
}

// Element i of the teacher's logits, of either type
template <class T>
__device__ __forceinline__ float ds_value(const DsArgs& a, int64_t i) {
  return a.t_f32 ? ((const float*)a.t)[i] : to_f(((const T*)a.t)[i]);
}

// 16 bytes at the address of any element: pieces lie at fixed places of a row, so that its sums do not
// depend on where it begins.
template <class T>
using Piece = Vec<T, kWide<T>>;
template <class T>
__device__ __forceinline__ Piece<T> ld_piece(const T* p) {
  Piece<T> x;
  __builtin_memcpy(&x, p, 16);
  return x;
}
template <class T>
__device__ __forceinline__ void st_piece(T* p, const Piece<T>& x) {
  __builtin_memcpy(p, &x, 16);
}

// The teacher's side of a row by one wave: its maximum and log2-sum, and the loss given the logits'.
template <class T>
__device__ __forceinline__ void ds_loss(const DsArgs& a, int64_t row, float zm, float l) {
  const int lane = threadIdx.x & 63;
  const T* z = (const T*)a.z + row * a.stride;
  float m = -INFINITY, s = 0.0f;
  for (int k = lane; k < a.K; k += 64) {
    const int64_t i = a.id[row * a.K + k];
    if (i >= 0 && i < a.V) ds_join(m, s, ds_value<T>(a, row * a.K + k), 1.0f, a.c);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ds_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), a.c);
  if (s != s) m = s;  // a NaN is an entry: it reaches the loss, also where it is the only one
  const bool some = s != 0.0f && m != -INFINITY;
  const float tl = __builtin_amdgcn_logf(s);
  float sum = 0.0f;
  for (int k = lane; k < a.K && some; k += 64) {
    const int64_t i = a.id[row * a.K + k];
    if (i < 0 || i >= a.V) continue;
    const float lp = __builtin_fmaf(ds_value<T>(a, row * a.K + k) - m, a.c, -tl);
    const float p = __builtin_amdgcn_exp2f(lp);
    if (p != 0.0f) sum += p * (lp - __builtin_fmaf(to_f(z[i]) - zm, a.c, -l));
  }
  sum = wave_sum_f(sum);
  if (lane == 0) {
    a.loss[row] = some ? a.tau * a.tau * kLn2 * sum : 0.0f;
    a.stats[row] = zm;
    a.stats[a.rows + row] = l;
    a.stats[2 * a.rows + row] = some ? m : -INFINITY;
    a.stats[3 * a.rows + row] = tl;
  }
}

template <class T, bool SPLIT>
__global__ __launch_bounds__(kDsThreads) void k_distill(DsArgs a) {
  constexpr int P = kWide<T>, U = 4;
  __shared__ float s_m[kDsThreads / 64], s_s[kDsThreads / 64];
  const int64_t row = SPLIT ? blockIdx.x / a.splits : blockIdx.x, part = SPLIT ? blockIdx.x % a.splits : 0;
  const int64_t v0 = part * a.len;
  const T* z = (const T*)a.z + row * a.stride + v0;
  const int n = (int)min(a.len, a.V - v0), pieces = n / P;
  float m = -INFINITY, s = 0.0f;
  auto take = [&](const float (&f)[P], int n) {
    float top = m;
#pragma unroll
    for (int j = 0; j < P; ++j) top = fmaxf(top, j < n ? f[j] : -INFINITY);
    const float at = top > -INFINITY ? top : 0.0f;
    s *= __builtin_amdgcn_exp2f((m - at) * a.c);
#pragma unroll
    for (int j = 0; j < P; ++j)
      if (j < n) s += __builtin_amdgcn_exp2f((f[j] - at) * a.c);
    m = top;
  };
  int i = threadIdx.x;
  for (; i + (U - 1) * kDsThreads < pieces; i += U * kDsThreads) {
    Piece<T> y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) y[u] = ld_piece(z + (int64_t)(i + u * kDsThreads) * P);
    float f[U][P], top = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < P; ++j) {
        f[u][j] = to_f(y[u].v[j]);
        top = fmaxf(top, f[u][j]);
      }
    const float at = top > -INFINITY ? top : 0.0f;
    s *= __builtin_amdgcn_exp2f((m - at) * a.c);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < P; ++j) s += __builtin_amdgcn_exp2f((f[u][j] - at) * a.c);
    m = top;
  }
  for (; i < pieces; i += kDsThreads) {
    const Piece<T> y = ld_piece(z + (int64_t)i * P);
    float f[P];
#pragma unroll
    for (int j = 0; j < P; ++j) f[j] = to_f(y.v[j]);
    take(f, P);
  }
  if (const int e = pieces * P + threadIdx.x; e < n) {
    const float f[P] = {to_f(z[e])};
    take(f, 1);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ds_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), a.c);
  if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = m, s_s[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  m = s_m[0], s = s_s[0];
#pragma unroll
  for (int w = 1; w < kDsThreads / 64; ++w) ds_join(m, s, s_m[w], s_s[w], a.c);
  if (SPLIT) {
    if (threadIdx.x == 0) {
      float* to = a.part + (row * a.splits + part) * 2;
      to[0] = m, to[1] = s;
    }
  } else {
    ds_loss<T>(a, row, m, __builtin_amdgcn_logf(s));
  }
}

// The parts of a row joined, one wave a row and one lane a part (48 rows of 21 parts: 3.7 us, one part after the
// other 5.5).
constexpr int kDsParts = 64;
template <class T>
__global__ __launch_bounds__(64) void k_distill_join(DsArgs a) {
  const int64_t row = blockIdx.x;
  const int i = threadIdx.x;
  const float* p = a.part + (row * a.splits + min(i, a.splits - 1)) * 2;
  float m = i < a.splits ? p[0] : -INFINITY, s = i < a.splits ? p[1] : 0.0f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ds_join(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), a.c);
  ds_loss<T>(a, row, m, __builtin_amdgcn_logf(s));
}

// dz of a part of a row, then the teacher's entries in it once more with their p.  An id may come several
// times; its p are summed in order by the first.  A bit for each place (modulo kDsBits) tells those that may
// come again, and only they look through the others (4096 x 32000 bf16: 16 entries a row 89 us, 64 92, 1024 177; with
// all looking 1024 took more than twice as long).
constexpr int kDsBits = 32768;
template <class T>
__global__ __launch_bounds__(kDsThreads) void k_distill_bwd(DsArgs a) {
  constexpr int P = kWide<T>, U = 4;
  extern __shared__ int s_id[];  // the teacher's ids of this part, as places in it (-1: none), then their p,
  float* s_p = (float*)(s_id + a.K);
  int* s_again = s_id + 2 * a.K;  // and those whose place may come again, n_again of them
  __shared__ unsigned s_once[kDsBits / 32], s_twice[kDsBits / 32];
  __shared__ int n_again;
  for (int b = threadIdx.x; b < kDsBits / 32; b += kDsThreads) s_once[b] = s_twice[b] = 0;
  if (threadIdx.x == 0) n_again = 0;
  const int64_t row = blockIdx.x / a.splits, v0 = blockIdx.x % a.splits * a.len;
  const T* z = (const T*)a.z + row * a.stride + v0;
  T* dz = (T*)a.dz + row * a.V + v0;
  const int n = (int)min(a.len, a.V - v0), pieces = n / P;
  const float zm = a.stats[row], l = a.stats[a.rows + row], tm = a.stats[2 * a.rows + row],
              tl = a.stats[3 * a.rows + row];
  const bool some = tm != -INFINITY;
  const float f = some ? a.g[row * a.g_stride] * a.tau : 0.0f;
  auto grad = [&](float y) { return some ? f * __builtin_amdgcn_exp2f(__builtin_fmaf(y - zm, a.c, -l)) : 0.0f; };
  auto put = [&](const Piece<T>& y, int i) {
    Piece<T> d;
#pragma unroll
    for (int j = 0; j < P; ++j) d.v[j] = from_f<T>(grad(to_f(y.v[j])));
    st_piece(dz + (int64_t)i * P, d);
  };
  int i = threadIdx.x;
  for (; i + (U - 1) * kDsThreads < pieces; i += U * kDsThreads) {
    Piece<T> y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) y[u] = ld_piece(z + (int64_t)(i + u * kDsThreads) * P);
#pragma unroll
    for (int u = 0; u < U; ++u) put(y[u], i + u * kDsThreads);
  }
  for (; i < pieces; i += kDsThreads) put(ld_piece(z + (int64_t)i * P), i);
  if (const int e = pieces * P + threadIdx.x; e < n) dz[e] = from_f<T>(grad(to_f(z[e])));
  if (!some) return;
  __syncthreads();  // the bits are clear
  for (int k = threadIdx.x; k < a.K; k += kDsThreads) {
    const int64_t id = a.id[row * a.K + k];
    const bool here = id >= v0 && id < v0 + n;
    const int e = here ? (int)(id - v0) : -1;
    s_id[k] = e;
    s_p[k] = here ? __builtin_amdgcn_exp2f(__builtin_fmaf(ds_value<T>(a, row * a.K + k) - tm, a.c, -tl)) : 0.0f;
    if (!here) continue;
    const unsigned bit = 1u << (e & 31), at = e % kDsBits / 32;
    if (atomicOr(&s_once[at], bit) & bit) atomicOr(&s_twice[at], bit);
  }
  __syncthreads();  // also the part's stores: its entries are written again with the teacher's part
  auto write = [&](int e, float p) {
    dz[e] = from_f<T>(f * (__builtin_amdgcn_exp2f(__builtin_fmaf(to_f(z[e]) - zm, a.c, -l)) - p));
  };
  for (int k = threadIdx.x; k < a.K; k += kDsThreads) {
    const int e = s_id[k];
    if (e < 0) continue;
    if (s_twice[e % kDsBits / 32] & (1u << (e & 31)))
      s_again[atomicAdd(&n_again, 1)] = k;
    else
      write(e, s_p[k]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_again; i += kDsThreads) {
    const int k = s_again[i], e = s_id[k];
    bool first = true;
    float p = 0.0f;
    for (int j = 0; j < a.K; ++j)
      if (s_id[j] == e) {
        first = first && j >= k;
        p += s_p[j];
      }
    if (first) write(e, p);
  }
}

static int ds_check(int dtype, int v_dtype, int64_t rows, int64_t V, int K, float tau) {
  if (!lm_dtype_ok(dtype) || (v_dtype != LSH_F32 && v_dtype != dtype) || !(tau > 0.0f) || !(tau < INFINITY))
    return LSH_ERR_ARG;
  if (rows < 0 || !lm_grid_ok(rows, kDsThreads) || V < 1 || V > 0x7fffffff / 2 || K < 0 || K > LSH_DISTILL_MAX_K)
    return LSH_ERR_SHAPE;
  return LSH_OK;
}

// Parts of a row: about 1024 workgroups, none of less than 4096 logits.
static int ds_splits(int64_t rows, int64_t V) {
  const int64_t most = std::min<int64_t>((V + 4095) / 4096, kDsParts);
  return (int)std::max<int64_t>(1, std::min(most, 1024 / std::max<int64_t>(rows, 1)));
}

static DsArgs ds_args(const void* logits, int64_t stride, int v_dtype, const void* values,
                      const int64_t* index, int64_t rows, int64_t V, int K, float tau) {
  DsArgs a = {};
  a.z = logits, a.stride = stride, a.t = values, a.t_f32 = v_dtype == LSH_F32, a.id = index;
  a.rows = rows, a.V = V, a.K = K;
  a.splits = ds_splits(rows, V);
  a.len = align_up((size_t)((V + a.splits - 1) / a.splits), 8);
  a.c = kLog2e / tau, a.tau = tau;
  return a;
}

}  // namespace lsh

using namespace lsh;

extern "C" size_t lsh_distill_workspace(int64_t rows, int64_t V) {
  if (ds_check(LSH_F32, LSH_F32, rows, V, 0, 1.0f)) return 0;
  const int splits = ds_splits(rows, V);
  return splits > 1 ? (size_t)rows * splits * 2 * sizeof(float) : 0;
}

extern "C" int lsh_distill_fwd(int dtype, const void* logits, int64_t stride, int v_dtype, const void* values,
                               const int64_t* index, float* loss, float* stats, int64_t rows, int64_t V,
                               int K, float tau, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = ds_check(dtype, v_dtype, rows, V, K, tau)) return rc;
  if (rows == 0) return LSH_OK;
  if (bad_ptr(logits) || (K > 0 && (bad_ptr(values) || bad_ptr(index))) || bad_ptr(loss) || bad_ptr(stats))
    return LSH_ERR_ARG;
  const size_t need = lsh_distill_workspace(rows, V);
  if (need && (bad_ptr(ws) || ws_bytes < need)) return LSH_ERR_WORKSPACE;
  DsArgs a = ds_args(logits, stride, v_dtype, values, index, rows, V, K, tau);
  a.loss = loss, a.stats = stats, a.part = (float*)ws;
  hipStream_t st = (hipStream_t)stream;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (a.splits > 1) {
      k_distill<T, true><<<dim3((unsigned)(rows * a.splits)), kDsThreads, 0, st>>>(a);
      k_distill_join<T><<<dim3((unsigned)rows), 64, 0, st>>>(a);
    } else {
      k_distill<T, false><<<dim3((unsigned)rows), kDsThreads, 0, st>>>(a);
    }
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" int lsh_distill_bwd(int dtype, const void* logits, int64_t stride, int v_dtype, const void* values,
                               const int64_t* index, const float* stats, const float* g, int64_t g_stride,
                               void* dlogits, int64_t rows, int64_t V, int K, float tau, void* stream) {
  if (int rc = ds_check(dtype, v_dtype, rows, V, K, tau)) return rc;
  if (rows == 0) return LSH_OK;
  if (bad_ptr(logits) || (K > 0 && (bad_ptr(values) || bad_ptr(index))) || bad_ptr(stats) || bad_ptr(g) ||
      bad_ptr(dlogits))
    return LSH_ERR_ARG;
  DsArgs a = ds_args(logits, stride, v_dtype, values, index, rows, V, K, tau);
  a.stats = (float*)stats, a.g = g, a.g_stride = g_stride, a.dz = dlogits;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_distill_bwd<T><<<dim3((unsigned)(rows * a.splits)), kDsThreads, (size_t)K * 12, (hipStream_t)stream>>>(a);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
