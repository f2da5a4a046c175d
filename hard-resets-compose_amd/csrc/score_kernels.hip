// Log probabilities of given tokens, the entropy of each row and its most likely alternatives.  With a temperature
// tau and z the logits,
//
//   p = softmax(z/tau),  logp = log p_y (0 where the row has no token y),  H = -sum_v p_v log p_v
//   top: the K largest logits, ties to the lower id, as log p and ids
//   dz_v = (g*([v = y] - p_v) - gH*p_v*(log p_v + H)) / tau       g, gH: gradients of logp and H; g is 0 without a token
//
// One pass over the logits holds the running maximum m, s = sum e and t = sum e*d, with d = (z - m)*c, e = 2^d and
// c = log2(e)/tau; then l = log2(s), log p = ln2*(d - l) and H = ln2*(l - t/s).  A logit of -inf has p = 0, and a row of
// nothing else has log p = -inf, H = 0 and no gradient.  A row with NaN or +inf has NaN.
//
// The K largest: each thread knows the largest of the logits that it read, and of its block of 4 pieces where that
// stands.  The K-th largest of those 256 is a bound that K logits reach, so only the few threads whose largest reaches it
// can hold one of the row's K: they read that block once more (others of theirs only if one of those reaches it too),
// and a handful more than K values come out, which are ranked by counting.  Values and ids are one whole number of 64
// bits, no two alike, so the order in which they are found does not matter.
#include <algorithm>
#include <type_traits>

#include "lsh_lm.h"

namespace lsh {

constexpr int kScThreads = 256, kScUnroll = 4, kScParts = 64;
constexpr float kScLog2e = 1.4426950408889634f, kScLn2 = 0.6931471805599453f;

struct ScArgs {
  const void* z;
  int64_t stride;
  const int64_t* token;
  float *logp, *entropy;
  float* stats;  // [3, rows]: m, l and H
  float* top_logp;
  int64_t* top_id;
  float* part;               // [rows, splits, 3]: m, s and t of each part
  unsigned long long* keys;  // [rows, splits, K]: each part's largest, in order
  const float *g, *gh;
  int64_t g_stride, gh_stride;
  void* dz;
  int64_t rows, V;
  int K, splits;
  int64_t len;  // logits of a part
  float c, tau;
};

// A value as a whole number in the same order, never 0; NaN before all, and one zero.
__device__ __forceinline__ unsigned sc_order(float x) {
  unsigned b = __builtin_bit_cast(unsigned, x + 0.0f);
  if (x != x) b = 0x7fc00000u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// A value and its id as a number: larger values first, then lower ids.
using Key = unsigned long long;
__device__ __forceinline__ Key sc_key(float x, unsigned id) { return (Key)sc_order(x) << 32 | (0xffffffffu - id); }
__device__ __forceinline__ unsigned sc_order(Key k) { return (unsigned)(k >> 32); }
__device__ __forceinline__ float sc_value(Key k) {
  const unsigned b = sc_order(k);
  return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ unsigned sc_id(Key k) { return 0xffffffffu - (unsigned)k; }

// (m, s, t) of two parts; a part without values has m = -inf, s = t = 0
__device__ __forceinline__ void sc_join(float& m, float& s, float& t, float m2, float s2, float t2, float c) {
  const float top = fmaxf(m, m2), at = top > -INFINITY ? top : 0.0f;
  const float d1 = fmaxf((m - at) * c, -1000.0f), d2 = fmaxf((m2 - at) * c, -1000.0f);
  const float e1 = __builtin_amdgcn_exp2f(d1), e2 = __builtin_amdgcn_exp2f(d2);
  t = e1 * __builtin_fmaf(d1, s, t) + e2 * __builtin_fmaf(d2, s2, t2);
  s = s * e1 + s2 * e2;
  m = top;
}

// 16 bytes at the address of any element
template <class T>
using ScPiece = Vec<T, kWide<T>>;
template <class T>
__device__ __forceinline__ ScPiece<T> sc_load(const T* p) {
  ScPiece<T> x;
  __builtin_memcpy(&x, p, 16);
  return x;
}

// The K largest of keys that the threads of a workgroup hold between them, in order, to out (0: none).  own: the value of
// a thread's largest, as sc_order (0: it has none); not known: the values of own are not to be relied on.
// scan(least, first, f) calls f with each key of the thread that is not less (and with some that are); first: its largest
// is enough, which has the value of least.  One call a kernel: its LDS is not shared.  NT threads, at least K.
template <int NT, class Scan, class Out>
__device__ __forceinline__ void sc_select(unsigned own, bool known, int K, Scan&& scan, Out&& out) {
  constexpr int LIST = 4 * NT;  // holds a key of each thread, too
  __shared__ unsigned s_value[NT], s_bound;
  __shared__ Key s_list[LIST], s_key;
  __shared__ int s_count, s_reach;
  const int tid = threadIdx.x;
  s_value[tid] = own;
  __syncthreads();
  if (tid < 64) {  // the K-th largest, bit by bit
    unsigned v[NT / 64], bound = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) v[i] = s_value[tid + 64 * i];
    int n = NT;  // threads that reach the bound
    for (unsigned bit = known ? 0x80000000u : 0; bit && n != K; bit >>= 1) {
      const unsigned t = bound | bit;
      int reach = 0;
#pragma unroll
      for (int i = 0; i < NT / 64; ++i) reach += __popcll(__ballot(v[i] >= t));
      if (reach >= K) bound = t, n = reach;
    }
    if (tid == 0) s_bound = bound, s_count = 0, s_reach = n;
  }
  __syncthreads();
  const unsigned bound = s_bound;
  bool mine = own && own >= bound;
  // The list of all keys that reach the bound.  Where many threads reach it, or the list does not hold them (long runs of
  // equal values, as where most of a row is masked): the K-th largest of the threads' largest keys, and the list of all
  // that reach that (2048 x 32000 bf16 with 20 alternatives, all but about ten masked: 83 us, by a list of all first 299).
  // Where it does not hold those either (a few threads hold most): the keys one after the other.  One place in the code
  // looks through a thread's keys for all of these: copies of it cost registers, and so waves.
  enum { kList, kLargest, kBounded, kNext } what = known && s_reach <= 2 * K + 32 ? kList : kLargest;
  Key least = (Key)bound << 32, last = ~(Key)0;
  for (int k = 0;;) {
    Key best = 0;
    if (mine) {
      const bool first = known && what == kLargest;
      scan(first ? (Key)own << 32 : least, first, [&](Key x) {
        if (what == kList || what == kBounded) {
          if (x < least) return;
          const int at = atomicAdd(&s_count, 1);
          if (at < LIST) s_list[at] = x;
        } else if (x < last) {
          best = max(best, x);
        }
      });
    }
    __syncthreads();
    if (what == kList || what == kBounded) {
      const int n = s_count;
      if (n <= LIST) {
        for (int i = tid; i < n; i += NT) {
          const Key x = s_list[i];
          int rank = 0;
          for (int j = 0; j < n; ++j) rank += s_list[j] > x;
          if (rank < K) out(rank, x);
        }
        for (int i = n + tid; i < K; i += NT) out(i, (Key)0);
        return;
      }
      what = what == kList ? kLargest : kNext;
    } else if (what == kLargest) {
      s_list[tid] = best;
      if (tid == 0) s_count = 0, s_key = 0;
      __syncthreads();
      int above = 0;
      for (int i = 0; i < NT; ++i) above += s_list[i] > best;
      if (above == K - 1 && best) s_key = best;
      __syncthreads();
      least = s_key;
      mine = best && best >= least;
      what = kBounded;
    } else {
      s_list[tid] = best;
      __syncthreads();
      for (int o = NT / 2; o > 0; o >>= 1) {
        if (tid < o) s_list[tid] = max(s_list[tid], s_list[tid + o]);
        __syncthreads();
      }
      last = s_list[0];
      __syncthreads();
      if (tid == 0) out(k, last);
      if (++k == K) return;
    }
  }
}

// What a row's statistics give: by one thread
// In natural logarithms, and z and m apart where their difference is no fp32 number: a logit at the lowest value of its
// type has a finite log p wherever fp32 has one.  With a finite z that needs a positive m, and below it z is -inf, as
// log p then is: m/tau, which may be -inf as well (the lowest value over 0.7), is not taken from it.
__device__ __forceinline__ float sc_logp(float z, float m, float l, float tau) {
  const float d = z - m;
  return l == -INFINITY ? -INFINITY : (d > -INFINITY ? d / tau : z / tau - fmaxf(m, 0.0f) / tau) - kScLn2 * l;
}
template <class T>
__device__ __forceinline__ void sc_finish(const ScArgs& a, int64_t row, float m, float s, float t) {
  const float l = __builtin_amdgcn_logf(s), H = s == 0.0f ? 0.0f : kScLn2 * (l - t / s);
  const int64_t y = a.token[row];
  const bool there = y >= 0 && y < a.V;
  a.logp[row] = there ? sc_logp(to_f(((const T*)a.z)[row * a.stride + y]), m, l, a.tau) : 0.0f;
  a.entropy[row] = H;
  if (a.stats) a.stats[row] = m, a.stats[a.rows + row] = l, a.stats[2 * a.rows + row] = H;
}
__device__ __forceinline__ void sc_put(const ScArgs& a, int64_t row, int k, Key key, float m, float l) {
  a.top_logp[row * a.K + k] = sc_logp(sc_value(key), m, l, a.tau);
  a.top_id[row * a.K + k] = sc_id(key);
}

// 8 waves a SIMD: while some workgroups select, others stream (2048 x 32000 bf16 with 5 alternatives: 38 us, with the 5
// waves that the compiler would leave 39, without alternatives 28).
template <class T, bool SPLIT, bool TOP, int NT>
__global__ __launch_bounds__(NT, 8) void k_score(ScArgs a) {
  constexpr int P = kWide<T>, U = kScUnroll, STEP = U * NT * P;
  __shared__ float s_stat[NT / 64][3];
  const int64_t row = SPLIT ? blockIdx.x / a.splits : blockIdx.x, part = SPLIT ? blockIdx.x % a.splits : 0;
  const int64_t v0 = part * a.len;
  const T* z = (const T*)a.z + row * a.stride + v0;
  const int n = (int)max((int64_t)0, min(a.len, a.V - v0));
  const int tid = threadIdx.x;
  // the first element of piece u of a thread in block b
  auto place = [&](int b, int u) { return b * STEP + (u * NT + tid) * P; };
  float m = -INFINITY, s = 0.0f, t = 0.0f;
  int best = 0;             // the block of the largest
  float other = -INFINITY;  // the largest of the other blocks
  auto take = [&](const float (&f)[U][P], int b) {
    float top = f[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < P; ++j) top = fmaxf(top, f[u][j]);
    if (TOP) {
      other = fmaxf(other, fminf(m, top));
      best = top > m ? b : best;
    }
    top = fmaxf(m, top);
    const float at = top > -INFINITY ? top : 0.0f;
    const float d0 = fmaxf((m - at) * a.c, -1000.0f), e0 = __builtin_amdgcn_exp2f(d0);
    t = e0 * __builtin_fmaf(d0, s, t);
    s *= e0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float d = (f[u][j] - at) * a.c, e = __builtin_amdgcn_exp2f(d);
        s += e;
        t = __builtin_fmaf(e, fmaxf(d, -1000.0f), t);
      }
    m = top;
  };
  const int whole = n / STEP;
  // where piece u of block b is read from: a piece that reaches over the end from P before the end on, so that no branch
  // stands around the loads.  What another thread reads too is left out.
  auto from = [&](int b, int u) { return b < whole || n < P ? place(b, u) : min(place(b, u), n - P); };
  auto read = [&](int b, float (&f)[U][P]) {
    ScPiece<T> y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) y[u] = sc_load(z + place(b, u));
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < P; ++j) f[u][j] = to_f(y[u].v[j]);
  };
  // what is left behind the whole blocks, -inf where nothing is
  auto read_rest = [&](int b, float (&f)[U][P]) {
    if (n >= P) {
      ScPiece<T> y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) y[u] = sc_load(z + from(b, u));
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < P; ++j) f[u][j] = from(b, u) + j >= place(b, u) ? to_f(y[u].v[j]) : -INFINITY;
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < P; ++j) f[u][j] = place(b, u) + j < n ? to_f(z[place(b, u) + j]) : -INFINITY;
    }
  };
  for (int b = 0; b < whole; ++b) {
    float f[U][P];
    read(b, f);
    take(f, b);
  }
  if (place(whole, 0) < n) {
    float f[U][P];
    read_rest(whole, f);
    take(f, whole);
  }
  const float mine = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    sc_join(m, s, t, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), __shfl_xor(t, o, 64), a.c);
  if ((tid & 63) == 0) s_stat[tid >> 6][0] = m, s_stat[tid >> 6][1] = s, s_stat[tid >> 6][2] = t;
  __syncthreads();
  m = s_stat[0][0], s = s_stat[0][1], t = s_stat[0][2];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) sc_join(m, s, t, s_stat[w][0], s_stat[w][1], s_stat[w][2], a.c);
  if (tid == 0) {
    if (SPLIT) {
      float* to = a.part + (row * a.splits + part) * 3;
      to[0] = m, to[1] = s, to[2] = t;
    } else {
      sc_finish<T>(a, row, m, s, t);
    }
  }
  if constexpr (TOP) {
    const int blocks = place(whole, 0) < n ? whole + 1 : whole;
    // the thread's keys of a block whose values reach a bound: which ones they are first, and then the few one by one
    auto block = [&](int b, unsigned bound, bool first, auto&& f) {
      const float least = sc_value((Key)bound << 32);
      float x[U][P];
      if (b < whole)
        read(b, x);
      else
        read_rest(b, x);
      unsigned long long there = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const int e = from(b, u) + j;
          // what is not less: also NaN, and any value where the bound is none
          if (!(x[u][j] < least) && e >= place(b, u) && e < n) there |= 1ull << (u * P + j);
        }
      if (first) there &= -there;  // of equal values the lowest id, which is the thread's largest key
      for (; there; there &= there - 1) {
        const int i = __ffsll((unsigned long long)there) - 1, e = from(b, i / P) + i % P;
        f(sc_key(to_f(z[e]), (unsigned)(v0 + e)));
      }
    };
    const float l = __builtin_amdgcn_logf(s);
    // a NaN, or +inf, in the row: the maxima leave NaN out
    const bool odd = s != s;
    sc_select<NT>(
        blocks ? sc_order(mine) : 0, !odd, a.K,
        [&](Key least, bool first, auto&& f) {
          const unsigned bound = least >> 32;
          const bool all = odd || (!first && sc_order(other) >= bound);
          const int b1 = all ? blocks : best + 1;
          for (int b = all ? 0 : best; b < b1; ++b)  // behind the id of least: what is larger
            block(b, bound + (!odd && v0 + (int64_t)b * STEP > (int64_t)sc_id(least)), first, f);
        },
        [&](int k, Key key) {
          if (SPLIT)
            a.keys[(row * a.splits + part) * a.K + k] = key;
          else
            sc_put(a, row, k, key, m, l);
        });
  }
}

// The parts of a row: a wave joins their statistics, and the workgroup their largest.
template <class T, bool TOP>
__global__ __launch_bounds__(kScThreads) void k_score_join(ScArgs a) {
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, i = tid & 63;
  const float* p = a.part + (row * a.splits + min(i, a.splits - 1)) * 3;
  float m = i < a.splits ? p[0] : -INFINITY, s = i < a.splits ? p[1] : 0.0f, t = i < a.splits ? p[2] : 0.0f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    sc_join(m, s, t, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), __shfl_xor(t, o, 64), a.c);
  if (tid == 0) sc_finish<T>(a, row, m, s, t);
  if constexpr (TOP) {
    const Key* keys = a.keys + row * a.splits * a.K;
    const int n = a.splits * a.K;
    unsigned own = 0;
    for (int k = tid; k < n; k += kScThreads) own = max(own, sc_order(keys[k]));
    const float l = __builtin_amdgcn_logf(s);
    sc_select<kScThreads>(
        own, true, a.K,
        [&](Key least, bool, auto&& f) {
          for (int k = tid; k < n; k += kScThreads)
            if (const Key x = keys[k]; x && x >= least) f(x);
        },
        [&](int k, Key key) { sc_put(a, row, k, key, m, l); });
  }
}

template <class T>
__global__ __launch_bounds__(kScThreads) void k_score_bwd(ScArgs a) {
  constexpr int P = kWide<T>, U = kScUnroll;
  const int64_t row = blockIdx.x / a.splits, v0 = blockIdx.x % a.splits * a.len;
  const T* z = (const T*)a.z + row * a.stride + v0;
  T* dz = (T*)a.dz + row * a.V + v0;
  const int n = (int)max((int64_t)0, min(a.len, a.V - v0)), pieces = n / P;
  const float m = a.stats[row], l = a.stats[a.rows + row], H = a.stats[2 * a.rows + row];
  const int64_t y = a.token[row];
  const bool some = l != -INFINITY, there = some && y >= 0 && y < a.V;
  const float per = 1.0f / a.tau;
  const float g = there ? a.g ? a.g[row * a.g_stride] * per : 0.0f : 0.0f;
  const float gh = some && a.gh ? a.gh[row * a.gh_stride] * per : 0.0f;
  const float flat = __builtin_fmaf(gh, H, g), slope = gh * kScLn2;
  const int at = there && y >= v0 && y < v0 + n ? (int)(y - v0) : -1;
  auto grad = [&](float v, int e) {
    float x = __builtin_fmaf(v - m, a.c, -l);
    x = x < -1000.0f ? -1000.0f : x;  // p = 0; a NaN stays
    const float d = -__builtin_amdgcn_exp2f(x) * __builtin_fmaf(slope, x, flat);
    return some ? e == at ? d + g : d : 0.0f;
  };
  auto put = [&](const ScPiece<T>& q, int i) {
    ScPiece<T> d;
#pragma unroll
    for (int j = 0; j < P; ++j) d.v[j] = from_f<T>(grad(to_f(q.v[j]), i * P + j));
    __builtin_memcpy(dz + (int64_t)i * P, &d, 16);
  };
  int i = threadIdx.x;
  for (; i + (U - 1) * kScThreads < pieces; i += U * kScThreads) {
    ScPiece<T> q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = sc_load(z + (int64_t)(i + u * kScThreads) * P);
#pragma unroll
    for (int u = 0; u < U; ++u) put(q[u], i + u * kScThreads);
  }
  for (; i < pieces; i += kScThreads) put(sc_load(z + (int64_t)i * P), i);
  if (const int e = pieces * P + threadIdx.x; e < n) dz[e] = from_f<T>(grad(to_f(z[e]), e));
}

static int sc_check(int dtype, int64_t rows, int64_t V, int K, float tau) {
  if (!lm_dtype_ok(dtype) || !(tau > 0.0f) || !(tau < INFINITY) || !(kScLog2e / tau < INFINITY)) return LSH_ERR_ARG;
  if (rows < 0 || !lm_grid_ok(rows, kScThreads) || V < 1 || V > 0x7fffffff / 2 || K < 0 || K > LSH_SCORE_MAX_TOP ||
      K > V)
    return LSH_ERR_SHAPE;
  return LSH_OK;
}

// Parts of a row: about 1024 workgroups, none of less than 4096 logits.
static int sc_splits(int64_t rows, int64_t V) {
  const int64_t most = std::min<int64_t>((V + 4095) / 4096, kScParts);
  return (int)std::max<int64_t>(1, std::min(most, 1024 / std::max<int64_t>(rows, 1)));
}

static ScArgs sc_args(const void* logits, int64_t stride, const int64_t* tokens, int64_t rows, int64_t V, int K,
                      float tau) {
  ScArgs a = {};
  a.z = logits, a.stride = stride, a.token = tokens, a.rows = rows, a.V = V, a.K = K;
  a.splits = sc_splits(rows, V);
  a.len = align_up((size_t)((V + a.splits - 1) / a.splits), 8);
  a.c = kScLog2e / tau, a.tau = tau;
  return a;
}

}  // namespace lsh

using namespace lsh;

extern "C" size_t lsh_score_workspace(int64_t rows, int64_t V, int K) {
  if (sc_check(LSH_F32, rows, V, K, 1.0f)) return 0;
  const int64_t splits = sc_splits(rows, V);
  return splits > 1 ? (size_t)(rows * splits) * (K * sizeof(Key) + 3 * sizeof(float)) : 0;
}

extern "C" int lsh_score_fwd(int dtype, const void* logits, int64_t stride, const int64_t* tokens, float* logp,
                             float* entropy, float* stats, float* top_logp, int64_t* top_index, int64_t rows,
                             int64_t V, int K, float tau, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = sc_check(dtype, rows, V, K, tau)) return rc;
  if (rows == 0) return LSH_OK;
  if (bad_ptr(logits) || bad_ptr(tokens) || bad_ptr(logp) || bad_ptr(entropy) ||
      (K > 0 && (bad_ptr(top_logp) || bad_ptr(top_index))))
    return LSH_ERR_ARG;
  const size_t need = lsh_score_workspace(rows, V, K);
  if (need && (bad_ptr(ws) || ws_bytes < need)) return LSH_ERR_WORKSPACE;
  ScArgs a = sc_args(logits, stride, tokens, rows, V, K, tau);
  a.logp = logp, a.entropy = entropy, a.stats = stats, a.top_logp = top_logp, a.top_id = top_index;
  a.keys = (Key*)ws, a.part = (float*)((Key*)ws + rows * a.splits * K);
  if (!lm_grid_ok(rows * a.splits, kScThreads)) return LSH_ERR_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto top) {
      constexpr bool TOP = decltype(top)::value;
      if (a.splits > 1) {
        k_score<T, true, TOP, kScThreads><<<dim3((unsigned)(rows * a.splits)), kScThreads, 0, st>>>(a);
        k_score_join<T, TOP><<<dim3((unsigned)rows), TOP ? kScThreads : 64, 0, st>>>(a);
      } else if (V <= 64 * kScUnroll * kWide<T> && K <= 32) {
        // one block of one wave, which waits for no others (8192 x 300 bf16 with 20 alternatives: 22 us, with four waves
        // 41); of more than half of its threads' largest the least is no bound to speak of
        k_score<T, false, TOP, 64><<<dim3((unsigned)rows), 64, 0, st>>>(a);
      } else {
        k_score<T, false, TOP, kScThreads><<<dim3((unsigned)rows), kScThreads, 0, st>>>(a);
      }
    };
    if (K > 0)
      go(std::true_type{});
    else
      go(std::false_type{});
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" int lsh_score_bwd(int dtype, const void* logits, int64_t stride, const int64_t* tokens, const float* stats,
                             const float* g_logp, int64_t g_stride, const float* g_entropy, int64_t ge_stride,
                             void* dlogits, int64_t rows, int64_t V, float tau, void* stream) {
  if (int rc = sc_check(dtype, rows, V, 0, tau)) return rc;
  if (rows == 0) return LSH_OK;
  if (bad_ptr(logits) || bad_ptr(tokens) || bad_ptr(stats) || bad_ptr(dlogits)) return LSH_ERR_ARG;
  ScArgs a = sc_args(logits, stride, tokens, rows, V, 0, tau);
  a.stats = (float*)stats, a.g = g_logp, a.g_stride = g_stride, a.gh = g_entropy, a.gh_stride = ge_stride;
  a.dz = dlogits;
  if (!lm_grid_ok(rows * a.splits, kScThreads)) return LSH_ERR_SHAPE;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_score_bwd<T><<<dim3((unsigned)(rows * a.splits)), kScThreads, 0, (hipStream_t)stream>>>(a);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
