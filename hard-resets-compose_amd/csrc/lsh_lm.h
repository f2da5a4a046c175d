// Device and host helpers shared by the language-model operators (linattn_kernels.hip,
// blocknorm_kernels.hip, embed_kernels.hip, distill_kernels.hip): element types, wide accesses and
// workgroup reductions.  Tensors are fp32, bf16 or fp16; every kernel computes in fp32 and rounds
// to the tensor's type where it stores, to nearest even.
#pragma once
#include "lsh_abi.h"
#include "lsh_common.h"

namespace lsh {

using bf16_t = __bf16;
using f16_t = _Float16;

// n consecutive elements as one access
template <class T, int n>
struct alignas(sizeof(T) * n) Vec {
  T v[n];
};

// elements of T in 16 bytes
template <class T>
constexpr int kWide = 16 / (int)sizeof(T);

template <class T>
__device__ __forceinline__ float to_f(T x) {
  return (float)x;
}
template <class T>
__device__ __forceinline__ T from_f(float x) {
  return (T)x;
}

inline bool lm_dtype_ok(int d) { return d == LSH_F32 || d == LSH_BF16 || d == LSH_F16; }
inline int lm_dtype_size(int d) { return d == LSH_F32 ? 4 : 2; }

// Whether a launch of so many workgroups fits: along an axis a grid has fewer than 2^32 threads.
inline bool lm_grid_ok(int64_t groups, int threads) { return groups < ((int64_t)1 << 32) / threads; }

// Calls f with a value of the C++ type of a dtype code.
template <class F>
inline void with_dtype(int d, F&& f) {
  if (d == LSH_F32)
    f(float{});
  else if (d == LSH_BF16)
    f(bf16_t{});
  else
    f(f16_t{});
}

// the value N lanes further in a row of 16
template <int N>
__device__ __forceinline__ float row_turned(float x) {
  const int i = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, i, 0x120 + N, 0xf, 0xf, true));
}

// The sum over a wave, the same in every lane: a tree within the rows of 16 lanes, then over the rows, all
// between registers.
__device__ __forceinline__ float wave_sum_f(float v) {
  v += row_turned<8>(v);
  v += row_turned<4>(v);
  v += row_turned<2>(v);
  v += row_turned<1>(v);
  const unsigned a = __builtin_bit_cast(unsigned, v);
  const auto x = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const unsigned x0 = x[0], x1 = x[1];
  v = __builtin_bit_cast(float, x0) + __builtin_bit_cast(float, x1);
  const unsigned b = __builtin_bit_cast(unsigned, v);
  const auto y = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  const unsigned y0 = y[0], y1 = y[1];
  return __builtin_bit_cast(float, y0) + __builtin_bit_cast(float, y1);
}

// V values of a row of D: WIDE the columns d, d + 1, ... in 16-byte accesses (D a multiple of V), otherwise
// the columns d, d + step, ... one by one, where lanes that are neighbours take neighbouring columns.
// Columns beyond D are read from the row's last ones, so that no branch stands around a wide load: behind a
// branch the compiler waits for each load before it issues the next.
template <int V, bool WIDE, class T>
struct Raw {
  static constexpr int P = V * sizeof(T) > 16 ? 16 / (int)sizeof(T) : V;
  Vec<T, P> x[V / P];
  __device__ __forceinline__ void load(const T* p, int d, int D, int step) {
    if constexpr (WIDE) {
      const int at = min(d, D - V);
#pragma unroll
      for (int i = 0; i < V / P; ++i) x[i] = *(const Vec<T, P>*)(p + at + i * P);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[j / P].v[j % P] = p[min(d + j * step, D - 1)];
    }
  }
  // as fp32, zeros beyond D or where `there` is false
  __device__ __forceinline__ void get(float (&f)[V], int d, int D, int step, bool there = true) const {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = there && d + (WIDE ? 0 : j * step) < D ? to_f(x[j / P].v[j % P]) : 0.0f;
  }
};
template <int V, bool WIDE, class T>
__device__ __forceinline__ void ld_vals(float (&f)[V], const T* p, int d, int D, int step) {
  Raw<V, WIDE, T> x;
  x.load(p, d, D, step);
  x.get(f, d, D, step);
}
template <int V, bool WIDE, class T>
__device__ __forceinline__ void st_vals(const float (&f)[V], T* p, int d, int D, int step) {
  if constexpr (WIDE) {
    if (d < D) {
      constexpr int P = V * sizeof(T) > 16 ? 16 / sizeof(T) : V;
#pragma unroll
      for (int i = 0; i < V; i += P) {
        Vec<T, P> x;
#pragma unroll
        for (int j = 0; j < P; ++j) x.v[j] = from_f<T>(f[i + j]);
        *(Vec<T, P>*)(p + d + i) = x;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (d + j * step < D) p[d + j * step] = from_f<T>(f[j]);
  }
}

}  // namespace lsh
