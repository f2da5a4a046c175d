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

__device__ __forceinline__ float wave_sum_f(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  return v;
}

}  // namespace lsh
