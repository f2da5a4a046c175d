// What stands between the projection of queries and keys and their attention: a norm of each head and its rotation
// by position, for all heads of a token in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w                      (without weights: y = x)
//   (y_i, y_j) -> (y_i cos - y_j sin, y_i sin + y_j cos)   angle = position * inv_freq[p] of pair p
//
// Pair p of the first `rot` columns is (p, p + rot/2), or the neighbours (2p, 2p + 1); the other columns pass.
// Gradients, with u those of y (the outputs' rotated back) and <.> the mean over the head:
//   m = u*w,  dx = r*(m - x*r^2*<m*x>),  dw = sum of u*x*r over tokens and heads,  r = 1/sqrt(mean(x^2) + eps)
//
// G lanes share a head, each with E pieces of V pairs, so a rotation needs no other lane and a norm a sum over G.  A
// wave takes a token's heads 64/G at a time and forms the angles once: in 64 bits down to a quarter turn (positions
// reach millions, and fp32 would keep a tenth of a radian there), then as Taylor sums in fp32.
#include <algorithm>
#include <type_traits>

#include "lsh_lm.h"

namespace lsh {

constexpr int kRtWaves = 4;

struct RtArgs {
  const void *q, *k;
  int64_t q_st, q_sb, q_sh, k_st, k_sb, k_sh;
  const int64_t* pos;
  int64_t p_st, p_sb;
  const double* freq;
  const float *wq, *wk;  // NULL: no norm
  float eps;
  void *qo, *ko;         // outputs, or the gradients of q and k; contiguous
  const void *gq, *gk;
  int64_t gq_st, gq_sb, gq_sh, gk_st, gk_sb, gk_sh;
  float* part;           // [grid, 2, D]: this workgroup's sums of dw
  int64_t B, items;
  int H, heads, D, rot, take, per_token;  // heads: of q and k together; take: of one item
};

// The sum over G neighbouring lanes, the same in each, between registers.
template <int CTRL>
__device__ __forceinline__ float rt_dpp(float x) {
  const int i = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, i, CTRL, 0xf, 0xf, true));
}
template <int G>
__device__ __forceinline__ float rt_sum(float v) {
  static_assert(G == 8 || G == 16 || G == 32, "lanes of a head");
  v += rt_dpp<0xb1>(v);   // lanes 1 0 3 2 of four
  v += rt_dpp<0x4e>(v);   // lanes 2 3 0 1
  v += rt_dpp<0x141>(v);  // the other four of eight
  if constexpr (G > 8) v += rt_dpp<0x140>(v);  // the other eight of sixteen
  if constexpr (G > 16) {
    const unsigned a = __builtin_bit_cast(unsigned, v);
    const auto x = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    const unsigned x0 = x[0], x1 = x[1];
    v = __builtin_bit_cast(float, x0) + __builtin_bit_cast(float, x1);
  }
  return v;
}

// cos and sin of position * freq.  Quarter turns are counted in 64 bits; what is left, at most pi/4, goes into
// Taylor sums whose next terms are below 2^-28.
__device__ __forceinline__ void rt_angle(double position, double freq, float& c, float& s) {
  const double turns = position * (freq * 0.63661977236758134308);  // quarters: 2 / pi
  const double whole = rint(turns);
  const float x = (float)((turns - whole) * 1.57079632679489661923);
  const int quarter = (int)(whole - 4.0 * floor(whole * 0.25));
  const float z = x * x;
  float ps = __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040);
  ps = __builtin_fmaf(z, ps, 1.0f / 120);
  ps = __builtin_fmaf(z, ps, -1.0f / 6);
  ps = __builtin_fmaf(x * z, ps, x);
  float pc = __builtin_fmaf(z, -1.0f / 3628800, 1.0f / 40320);
  pc = __builtin_fmaf(z, pc, -1.0f / 720);
  pc = __builtin_fmaf(z, pc, 1.0f / 24);
  pc = __builtin_fmaf(z, pc, -0.5f);
  pc = __builtin_fmaf(z, pc, 1.0f);
  const float a = quarter & 1 ? ps : pc, b = quarter & 1 ? pc : ps;
  c = (quarter + 1) & 2 ? -a : a;
  s = quarter & 2 ? -b : b;
}

// 1/sqrt(x): the instruction (1 ulp) where neither side leaves the normal numbers.
__device__ __forceinline__ float rt_rsqrt(float x) {
  return x > 0x1p-100f && x < 0x1p100f ? __builtin_amdgcn_rsqf(x) : 1.0f / sqrtf(x);
}

// The columns of a lane's E pieces and how its 2*V values pair up: (j, V + j), or neighbours.
template <int V, int G, int E, bool NEXT>
struct RtLane {
  int lo[E], hi[E], pair[E];
  bool there[E];
  __device__ __forceinline__ RtLane(const RtArgs& a) {
    const int slot = threadIdx.x % G, half = a.rot / 2;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int p = (e * G + slot) * V;
      there[e] = p < a.D / 2;
      pair[e] = p;
      if (!there[e])
        lo[e] = hi[e] = 0;
      else if (NEXT)
        lo[e] = 2 * p, hi[e] = 2 * p + V;
      else if (p < half)
        lo[e] = p, hi[e] = p + half;
      else
        lo[e] = half + p, hi[e] = half + p + (a.D / 2 - half);
    }
  }
  // Whether pair j of piece e turns.  The others are left alone: times a sine of 0 an infinity or a NaN in one column
  // would reach the other.
  __device__ __forceinline__ bool turns(const RtArgs& a, int e, int j) const { return pair[e] + j < a.rot / 2; }
  static __device__ __forceinline__ constexpr int first(int j) { return NEXT ? 2 * j : j; }
  static __device__ __forceinline__ constexpr int second(int j) { return NEXT ? 2 * j + 1 : V + j; }
  template <class T>
  __device__ __forceinline__ void load(const T* p, Vec<T, V> (&x)[E][2]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e][0] = *(const Vec<T, V>*)(p + lo[e]), x[e][1] = *(const Vec<T, V>*)(p + hi[e]);
  }
  // as fp32; where there are no columns, some others of the head
  template <class T>
  static __device__ __forceinline__ void get(const Vec<T, V> (&x)[E][2], float (&f)[E][2 * V]) {
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int j = 0; j < V; ++j) f[e][j] = to_f(x[e][0].v[j]), f[e][V + j] = to_f(x[e][1].v[j]);
  }
  // the sum over a head of the products a*b
  __device__ __forceinline__ float dot(const float (&a)[E][2 * V], const float (&b)[E][2 * V]) const {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) s = __builtin_fmaf(a[e][j], b[e][j], s);
      sum += there[e] ? s : 0.0f;
    }
    return rt_sum<G>(sum);
  }
  template <class T>
  __device__ __forceinline__ void put(T* p, const float (&f)[E][2 * V]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      Vec<T, V> u, v;
#pragma unroll
      for (int j = 0; j < V; ++j) u.v[j] = from_f<T>(f[e][j]), v.v[j] = from_f<T>(f[e][V + j]);
      if (there[e]) *(Vec<T, V>*)(p + lo[e]) = u, *(Vec<T, V>*)(p + hi[e]) = v;
    }
  }
  __device__ __forceinline__ void weights(const float* w, float (&f)[E][2 * V]) const {
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int j = 0; j < V; ++j) f[e][j] = w[lo[e] + j], f[e][V + j] = w[hi[e] + j];
  }
};

// 8192 tokens of 16 + 4 heads of 128, bf16: forward 22 us for 84 MB (3.8 TB/s), gradients 31 us for 126 MB (4.1 TB/s)
// and 4 for the weights' sums.  What bounds them: a wave's loads, its sums over lanes and its stores follow one
// another, and registers leave 8 waves a SIMD forwards and 5 backwards to cover that.  (Copies of the work for heads of
// q alone, of k alone and of either save the choice of weights, an instruction in ten, and cost the fifth wave: 34.)
template <class T, int V, int G, int E, bool NEXT, bool BWD>
__global__ __launch_bounds__(kRtWaves * 64, 5) void k_rotate(RtArgs a) {
  using Lane = RtLane<V, G, E, NEXT>;
  using Row = float[E][2 * V];
  __shared__ float s_sum[BWD ? kRtWaves : 1][BWD ? 2 * 2 * V * E * G : 1];
  const Lane at(a);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = (threadIdx.x & 63) / G;
  const bool norm = a.wq != nullptr;
  const float per = 1.0f / a.D;
  Row wq, wk, sq = {}, sk = {};
  if (norm) at.weights(a.wq, wq), at.weights(a.wk, wk);
  for (int64_t item = (int64_t)blockIdx.x * kRtWaves + wave; item < a.items; item += (int64_t)gridDim.x * kRtWaves) {
    const int64_t token = item / a.per_token, t = token / a.B, b = token - t * a.B;
    const int head0 = (int)(item - token * a.per_token) * a.take, head1 = min(a.heads, head0 + a.take);
    float c[E][V], s[E][V];
    const double position = a.rot ? (double)a.pos[t * a.p_st + b * a.p_sb] : 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        c[e][j] = 1.0f, s[e][j] = 0.0f;
        if (at.turns(a, e, j)) rt_angle(position, a.freq[at.pair[e] + j], c[e][j], s[e][j]);
      }
    for (int h = head0; h < head1; h += 64 / G) {
      const bool live = h + sub < head1;
      const int head = live ? h + sub : head1 - 1;
      const bool is_q = head < a.H;
      const int own = is_q ? head : head - a.H;  // the head's number among those of q, or k
      T* out = (T*)(is_q ? a.qo : a.ko) + (token * (is_q ? a.H : a.heads - a.H) + own) * a.D;
      Vec<T, V> rx[E][2], rg[E][2];
      if (!BWD || norm)
        at.load((const T*)(is_q ? a.q : a.k) +
                    (is_q ? t * a.q_st + b * a.q_sb + own * a.q_sh : t * a.k_st + b * a.k_sb + own * a.k_sh),
                rx);
      if (BWD)
        at.load((const T*)(is_q ? a.gq : a.gk) +
                    (is_q ? t * a.gq_st + b * a.gq_sb + own * a.gq_sh : t * a.gk_st + b * a.gk_sb + own * a.gk_sh),
                rg);
      Row w, f, y;
      if (norm)
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) w[e][j] = is_q ? wq[e][j] : wk[e][j];
      if constexpr (!BWD) {
        at.get(rx, f);
        if (norm) {
          const float r = rt_rsqrt(at.dot(f, f) * per + a.eps);
#pragma unroll
          for (int e = 0; e < E; ++e)
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) f[e][j] *= r * w[e][j];
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float u = f[e][Lane::first(j)], v = f[e][Lane::second(j)];
            y[e][Lane::first(j)] = at.turns(a, e, j) ? __builtin_fmaf(u, c[e][j], -(v * s[e][j])) : u;
            y[e][Lane::second(j)] = at.turns(a, e, j) ? __builtin_fmaf(u, s[e][j], v * c[e][j]) : v;
          }
      } else {
        at.get(rg, y);
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float u = y[e][Lane::first(j)], v = y[e][Lane::second(j)];
            y[e][Lane::first(j)] = at.turns(a, e, j) ? __builtin_fmaf(u, c[e][j], v * s[e][j]) : u;
            y[e][Lane::second(j)] = at.turns(a, e, j) ? __builtin_fmaf(v, c[e][j], -(u * s[e][j])) : v;
          }
        if (norm) {
          at.get(rx, f);
          const float r = rt_rsqrt(at.dot(f, f) * per + a.eps);
          const bool to_q = live && is_q, to_k = live && !is_q;
#pragma unroll
          for (int e = 0; e < E; ++e)
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
              const float x = y[e][j] * f[e][j];  // chosen and not multiplied by 0: a NaN stays in its own sum
              sq[e][j] = to_q ? __builtin_fmaf(x, r, sq[e][j]) : sq[e][j];
              sk[e][j] = to_k ? __builtin_fmaf(x, r, sk[e][j]) : sk[e][j];
              y[e][j] *= w[e][j];
            }
          const float back = r * r * (at.dot(y, f) * per);
#pragma unroll
          for (int e = 0; e < E; ++e)
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) y[e][j] = r * __builtin_fmaf(-f[e][j], back, y[e][j]);
        }
      }
      if (live) at.put(out, y);
    }
  }
  if constexpr (BWD) {
    if (!norm) return;
    // the heads that the wave's lanes held side by side, then the waves
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) {
        float u = sq[e][j], v = sk[e][j];
#pragma unroll
        for (int o = G; o < 64; o *= 2) u += __shfl_xor(u, o, 64), v += __shfl_xor(v, o, 64);
        if (sub == 0 && at.there[e]) {
          const int col = j < V ? at.lo[e] + j : at.hi[e] + j - V;
          s_sum[wave][col] = u, s_sum[wave][a.D + col] = v;
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += kRtWaves * 64) {
      float sum = s_sum[0][i];
#pragma unroll
      for (int w = 1; w < kRtWaves; ++w) sum += s_sum[w][i];
      a.part[(int64_t)blockIdx.x * 2 * a.D + i] = sum;
    }
  }
}

// The workgroups' sums of dw: kRtRuns runs of workgroups at once, each as 8 sums, and pairs of those and of the runs.  One
// after the other the up to 40 of a run and then the runs drift: equal terms are off by up to 14 * 2^-24 of their sum.
constexpr int kRtCols = 32, kRtRuns = 32;
__global__ __launch_bounds__(kRtCols* kRtRuns) void k_rotate_sums(const float* __restrict__ part, int P, int D,
                                                                  float* dwq, float* dwk) {
  __shared__ float s_run[kRtRuns][kRtCols];
  const int c = threadIdx.x % kRtCols, run = threadIdx.x / kRtCols, i = blockIdx.x * kRtCols + c;
  const int per = (P + kRtRuns - 1) / kRtRuns, p1 = min(P, (run + 1) * per);
  float s[8] = {};
  if (i < 2 * D) {
    const size_t row = 2 * D;
    const float* at = part + run * per * row + i;
    int p = run * per;
#pragma unroll 2
    for (; p + 8 <= p1; p += 8, at += 8 * row)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += at[j * row];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (p + j < p1) s[j] += at[j * row];
  }
#pragma unroll
  for (int n = 4; n > 0; n /= 2)
#pragma unroll
    for (int j = 0; j < n; ++j) s[j] += s[j + n];
  s_run[run][c] = s[0];
  __syncthreads();
  if (run != 0 || i >= 2 * D) return;
  float r[kRtRuns];
#pragma unroll
  for (int j = 0; j < kRtRuns; ++j) r[j] = s_run[j][c];
#pragma unroll
  for (int n = kRtRuns / 2; n > 0; n /= 2)
#pragma unroll
    for (int j = 0; j < n; ++j) r[j] += r[j + n];
  float* out = i < D ? dwq : dwk;
  if (out) out[i % D] = r[0];
}

// reads: whether q and k are read (the gradients of a rotation alone do without)
static int rt_check(const lsh_rotate* a, bool reads) {
  if (!a || !lm_dtype_ok(a->dtype) || !(a->eps >= 0.0f) || !a->q_weight != !a->k_weight) return LSH_ERR_ARG;
  const int64_t most = (int64_t)1 << 40;
  if (a->T < 0 || a->B < 0 || a->H < 0 || a->HK < 0 || a->H > 0x10000 || a->HK > 0x10000 || a->D < 2 || a->D % 2 ||
      a->D > LSH_ROTATE_MAX_D || a->rot < 0 || a->rot % 2 || a->rot > a->D || a->T > most || a->B > most ||
      (a->T > 0 && a->B > most / a->T))
    return LSH_ERR_SHAPE;
  const bool some = a->T > 0 && a->B > 0;
  if (some && ((reads && a->H > 0 && bad_ptr(a->q)) || (reads && a->HK > 0 && bad_ptr(a->k)) ||
               (a->rot > 0 && (bad_ptr(a->positions) || bad_ptr(a->inv_freq)))))
    return LSH_ERR_ARG;
  return LSH_OK;
}

static RtArgs rt_args(const lsh_rotate* p) {
  RtArgs a = {};
  a.q = p->q, a.k = p->k;
  a.q_st = p->q_st, a.q_sb = p->q_sb, a.q_sh = p->q_sh, a.k_st = p->k_st, a.k_sb = p->k_sb, a.k_sh = p->k_sh;
  a.pos = p->positions, a.p_st = p->p_st, a.p_sb = p->p_sb, a.freq = p->inv_freq;
  a.wq = p->q_weight, a.wk = p->k_weight, a.eps = p->eps;
  a.B = p->B, a.H = (int)p->H, a.heads = (int)(p->H + p->HK), a.D = p->D, a.rot = p->rot;
  return a;
}

// Whether pieces of four lie at multiples of their size and never across the end of what is rotated.
static bool rt_wide(const RtArgs& a, int size, bool next) {
  if (next ? a.D % 8 || a.rot % 2 : a.D % 8 || a.rot % 8) return false;
  for (const void* p : {a.q, a.k, (const void*)a.qo, (const void*)a.ko, a.gq, a.gk})
    if ((uintptr_t)p % (4 * size)) return false;
  for (int64_t s : {a.q_st, a.q_sb, a.q_sh, a.k_st, a.k_sb, a.k_sh, a.gq_st, a.gq_sb, a.gq_sh, a.gk_st, a.gk_sb, a.gk_sh})
    if (s % 4) return false;
  return true;
}

// Calls f with the pairs of a piece, the lanes of a head and the pieces of a lane.
template <class F>
static void with_head(bool wide, int D, F&& f) {
  using std::integral_constant;
  const integral_constant<int, 1> one;
  const integral_constant<int, 32> half;
  if (wide && D <= 64)
    f(integral_constant<int, 4>{}, integral_constant<int, 8>{}, one);
  else if (wide && D <= 128)
    f(integral_constant<int, 4>{}, integral_constant<int, 16>{}, one);
  else if (wide)
    f(integral_constant<int, 4>{}, half, one);
  else if (D <= 64)
    f(one, half, one);
  else if (D <= 128)
    f(one, half, integral_constant<int, 2>{});
  else
    f(one, half, integral_constant<int, 4>{});
}

// Workgroups of the gradients, each with 2*D sums of its own: as many as the chip holds at once with 5 waves a SIMD
// (8192 x 20 heads of 128 bf16: 31 us, with 1024 or 2048 34).
constexpr int64_t kRtMost = 256 * 5;

// Launches a pass; *grid: its workgroups.  False: too many.
template <bool BWD>
static bool rt_launch(RtArgs& a, int dtype, int64_t tokens, bool next, hipStream_t st, int64_t* grid) {
  const bool wide = rt_wide(a, lm_dtype_size(dtype), next);
  bool fits = true;
  with_head(wide, a.D, [&](auto v, auto g, auto e) {
    constexpr int V = decltype(v)::value, G = decltype(g)::value, E = decltype(e)::value;
    // an item is as many of a token's heads as leave 8192 waves something to do: its angles are formed once
    const int64_t turns = (a.heads + 64 / G - 1) / (64 / G);
    const int64_t split = std::min(turns, std::max<int64_t>(1, (8192 + tokens - 1) / tokens));
    a.take = (int)((turns + split - 1) / split) * (64 / G);
    a.per_token = (a.heads + a.take - 1) / a.take;
    a.items = tokens * a.per_token;
    *grid = (a.items + kRtWaves - 1) / kRtWaves;
    if (BWD) *grid = std::min(*grid, kRtMost);
    fits = lm_grid_ok(*grid, kRtWaves * 64);
    if (!fits) return;
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      if (next)
        k_rotate<T, V, G, E, true, BWD><<<dim3((unsigned)*grid), kRtWaves * 64, 0, st>>>(a);
      else
        k_rotate<T, V, G, E, false, BWD><<<dim3((unsigned)*grid), kRtWaves * 64, 0, st>>>(a);
    });
  });
  return fits;
}

}  // namespace lsh

using namespace lsh;

extern "C" int lsh_rotate_fwd(const lsh_rotate* p, void* q_out, void* k_out, void* stream) {
  if (int rc = rt_check(p, true)) return rc;
  if (p->T == 0 || p->B == 0 || p->H + p->HK == 0) return LSH_OK;
  if ((p->H > 0 && bad_ptr(q_out)) || (p->HK > 0 && bad_ptr(k_out))) return LSH_ERR_ARG;
  RtArgs a = rt_args(p);
  a.qo = q_out, a.ko = k_out;
  int64_t grid;
  if (!rt_launch<false>(a, p->dtype, p->T * p->B, p->neighbours != 0, (hipStream_t)stream, &grid)) return LSH_ERR_SHAPE;
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" size_t lsh_rotate_bwd_workspace(const lsh_rotate* p) {
  if (rt_check(p, false) || !p->q_weight) return 0;
  return (size_t)kRtMost * 2 * p->D * sizeof(float);
}

extern "C" int lsh_rotate_bwd(const lsh_rotate* p, const void* gq, int64_t gq_st, int64_t gq_sb, int64_t gq_sh,
                              const void* gk, int64_t gk_st, int64_t gk_sb, int64_t gk_sh, void* dq, void* dk,
                              float* dq_weight, float* dk_weight, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = rt_check(p, p && p->q_weight)) return rc;
  const bool some = p->T > 0 && p->B > 0 && p->H + p->HK > 0;
  hipStream_t st = (hipStream_t)stream;
  int64_t grid = 0;
  const size_t need = lsh_rotate_bwd_workspace(p);
  if (some) {
    if ((p->H > 0 && (bad_ptr(gq) || bad_ptr(dq))) || (p->HK > 0 && (bad_ptr(gk) || bad_ptr(dk)))) return LSH_ERR_ARG;
    if (need && (bad_ptr(ws) || ws_bytes < need)) return LSH_ERR_WORKSPACE;
    RtArgs a = rt_args(p);
    a.qo = dq, a.ko = dk, a.gq = gq, a.gk = gk, a.part = (float*)ws;
    a.gq_st = gq_st, a.gq_sb = gq_sb, a.gq_sh = gq_sh, a.gk_st = gk_st, a.gk_sb = gk_sb, a.gk_sh = gk_sh;
    if (!rt_launch<true>(a, p->dtype, p->T * p->B, p->neighbours != 0, st, &grid)) return LSH_ERR_SHAPE;
    LSH_CHECK_LAUNCH();
  }
  if (p->q_weight && (dq_weight || dk_weight)) {
    k_rotate_sums<<<dim3((2 * p->D + kRtCols - 1) / kRtCols), kRtCols * kRtRuns, 0, st>>>(
        (const float*)ws, (int)grid, p->D, dq_weight, dk_weight);
    LSH_CHECK_LAUNCH();
  }
  return LSH_OK;
}
