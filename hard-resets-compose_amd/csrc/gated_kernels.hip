// A gated linear recurrence: a leaky integrator whose decay is another one for each channel and token,
//
//   a_t = sigmoid(gate_t), or exp(min(gate_t, 0))        in [0, 1]
//   h_t = a_t*h_{t-1} + w_t*x_t,  w_t = 1 - a_t or 1      (h_{t-1} dropped where a sequence starts)
//
// and its gradients, with E the adjoint of h and F_t = a_t*E_t (0 where a sequence starts) what goes back:
//   E_t = dh_t + F_{t+1},  F_T = dh_end,  dh0 = F_0
//   dx_t = w_t*E_t,  dgate_t = E_t*(h_{t-1} - [w = 1 - a]*x_t)*da/dgate
//
// A step is an affine map, and so is a run of steps: (P, H) with h_end = P*h_begin + H, and backwards (P, Q) with
// F_begin = P*F_end + Q and the same P.  A lane has V neighbouring channels, a wave kGsR rows of them in registers,
// and a workgroup's waves hold consecutive rows: the waves' maps meet in LDS, each wave composes those before its own,
// and then writes its rows from the state before them.  Where there are too few channels for the chip the rows are cut
// into segments, whose maps an extra pass over the operands forms.  The gradients take h_{t-1} from the state before
// every kGsRows rows, which the forward keeps in fp32, and form it again: h itself may have 16 bits.
//
// A start is a factor -0 (decays are never negative): a marked product stays marked and drops what it is
// applied to, also an infinity or a NaN.
#include <algorithm>
#include <type_traits>

#include "lsh_lm.h"

namespace lsh {

constexpr int kGsR = 16, kGsW = 8, kGsRows = kGsR * kGsW;

struct GsArgs {
  const void *x, *g;
  int64_t x_st, x_sb, g_st, g_sb;
  const uint8_t* starts;  // [T, B], or NULL
  const float* h0;        // [n], or NULL
  void* h;
  float *h_end, *saved;   // saved: [ceil(T / kGsRows), n], or NULL
  const void* dh;
  int64_t d_st, d_sb;
  const float* d_end;
  void *dx, *dg;
  float* dh0;
  float* part;            // [S, 2, n]: the segments' maps
  int64_t T, B, D, n, pieces, len;  // n = B*D channels in pieces of V; rows of a segment
  int groups, S, sigmoid, mix;
};

// e^x for x <= 0: the hardware's power of two with what the product x*log2(e) loses put back
__device__ __forceinline__ float gs_exp(float x) {
  x = x < -150.0f ? -150.0f : x;  // 0, and no inf - inf; a NaN stays
  constexpr float kHi = 1.44269502f, kLo = 1.92596299e-8f;  // log2(e)
  const float t = x * kHi, r = __builtin_fmaf(x, kHi, -t) + x * kLo;
  const float y = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(y, r * 0.693147181f, y);
}

// (a, 1 - a).  Of a sigmoid the smaller one is e/(1 + e) with e = exp(-|g|), 1 - e^g is a Taylor sum where it would
// cancel, and a decay near one is what is left of one: it is raised to hundreds of rows, so it is rounded once (with
// the hardware's 1/(1 + e) and 2^x in its place the results of 1000 rows in fp32 were off by 7.2e-7 of their norm, so 2.2e-7).
__device__ __forceinline__ void gs_gate(int sigmoid, float g, float& a, float& w) {
  if (sigmoid) {
    const float e = gs_exp(-__builtin_fabsf(g)), s = e * __builtin_amdgcn_rcpf(1.0f + e), r = 1.0f - s;
    a = g >= 0.0f ? r : s;
    w = g >= 0.0f ? s : r;
  } else {
    g = g > 0.0f ? 0.0f : g;
    float p = __builtin_fmaf(g, 1.0f / 5040, 1.0f / 720);
    p = __builtin_fmaf(g, p, 1.0f / 120);
    p = __builtin_fmaf(g, p, 1.0f / 24);
    p = __builtin_fmaf(g, p, 1.0f / 6);
    p = __builtin_fmaf(g, p, 0.5f);
    p = __builtin_fmaf(g, p, 1.0f);
    const float e = gs_exp(g);
    w = g > -0.35f ? -g * p : 1.0f - e;
    a = g > -0.35f ? 1.0f - w : e;
  }
}

constexpr unsigned kGsStart = 0x80000000u;  // the factor of a start
__device__ __forceinline__ bool gs_marked(float p) { return __builtin_bit_cast(unsigned, p) == kGsStart; }
template <bool MASK>
__device__ __forceinline__ float gs_apply(float p, float h, float before) {
  const float y = __builtin_fmaf(p, before, h);
  return MASK && gs_marked(p) ? h : y;
}
template <bool MASK>
__device__ __forceinline__ float gs_product(float first, float then) {
  return MASK && gs_marked(then) ? then : MASK && gs_marked(first) ? first : first * then;
}

// A lane's channels
template <class T, int V>
struct GsLane {
  bool there;
  int64_t c, b, x_at, g_at, d_at;  // the first channel, its batch, and where they lie in a row
  __device__ __forceinline__ GsLane(const GsArgs& a, int group) {
    const int64_t p = (int64_t)group * 64 + (threadIdx.x & 63);
    there = p < a.pieces;
    c = (there ? p : a.pieces - 1) * V;
    b = c / a.D;
    const int64_t d = c - b * a.D;
    x_at = b * a.x_sb + d, g_at = b * a.g_sb + d, d_at = b * a.d_sb + d;
  }
};

// kGsR rows of a lane as read; rows from `end` on are read from the one before it
template <class T, int V>
struct GsRows {
  Vec<T, V> v[kGsR];
  __device__ __forceinline__ void load(const T* p, int64_t stride, int64_t t, int64_t end) {
    if (t + kGsR <= end) {
      p += t * stride;
#pragma unroll
      for (int i = 0; i < kGsR; ++i) v[i] = *(const Vec<T, V>*)(p + i * stride);
    } else {
#pragma unroll
      for (int i = 0; i < kGsR; ++i) {
        const int64_t at = t + i < end ? t + i : end - 1;
        v[i] = *(const Vec<T, V>*)(p + at * stride);
      }
    }
  }
};
struct GsStarts {
  uint8_t v[kGsR];
  __device__ __forceinline__ void load(const GsArgs& a, int64_t b, int64_t t, int64_t end) {
#pragma unroll
    for (int i = 0; i < kGsR; ++i) v[i] = a.starts[(t + i < end ? t + i : end - 1) * a.B + b];
  }
};

// Where segments are needed: the map of each, forwards (x, gate) or backwards (gate, dh).  A wave takes its share of the
// segment's rows, its map in registers.
template <class T, int V, bool MASK, bool BWD>
__global__ __launch_bounds__(kGsW * 64) void k_gated_sums(GsArgs a) {
  __shared__ float s_map[kGsW][2][64 * V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = blockIdx.x % a.groups, seg = blockIdx.x / a.groups;
  const GsLane<T, V> at(a, group);
  const T* x = BWD ? (const T*)a.dh + at.d_at : (const T*)a.x + at.x_at;
  const int64_t x_st = BWD ? a.d_st : a.x_st;
  const T* g = (const T*)a.g + at.g_at;
  const int64_t t1 = min(a.T, (seg + 1) * a.len);
  const int64_t per = a.len / kGsW, lo = seg * a.len + wave * per, hi = min(t1, lo + per);
  float P[V], H[V];
#pragma unroll
  for (int j = 0; j < V; ++j) P[j] = 1.0f, H[j] = 0.0f;
  const bool zeros = BWD && !a.dh;
  for (int64_t k = lo; k < hi; k += kGsR) {
    const int64_t t = BWD ? lo + (hi - lo - 1) / kGsR * kGsR - (k - lo) : k;
    GsRows<T, V> rx, rg;
    GsStarts rs;
    if (!zeros) rx.load(x, x_st, t, hi);
    rg.load(g, a.g_st, t, hi);
    if (MASK) rs.load(a, at.b, t, hi);
#pragma unroll
    for (int n = 0; n < kGsR; ++n) {
      const int i = BWD ? kGsR - 1 - n : n;
      if (t + i >= hi) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float f, w;
        gs_gate(a.sigmoid, to_f(rg.v[i].v[j]), f, w);
        if (MASK && rs.v[i]) f = __builtin_bit_cast(float, kGsStart);
        if constexpr (BWD) {
          const float d = zeros ? 0.0f : to_f(rx.v[i].v[j]);
          H[j] = MASK && gs_marked(f) ? 0.0f : f * (d + H[j]);
        } else {
          const float v = to_f(rx.v[i].v[j]);
          H[j] = gs_apply<MASK>(f, a.mix ? w * v : v, H[j]);
        }
        P[j] = gs_product<MASK>(P[j], f);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) s_map[wave][0][lane * V + j] = P[j], s_map[wave][1][lane * V + j] = H[j];
  __syncthreads();
  if (wave != 0 || !at.there) return;
#pragma unroll
  for (int j = 0; j < V; ++j) P[j] = 1.0f, H[j] = 0.0f;
  for (int n = 0; n < kGsW; ++n) {
    const int w = BWD ? kGsW - 1 - n : n;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float p = s_map[w][0][lane * V + j];
      H[j] = gs_apply<MASK>(p, s_map[w][1][lane * V + j], H[j]);
      P[j] = gs_product<MASK>(P[j], p);
    }
  }
  float* out = a.part + (int64_t)seg * 2 * a.n + at.c;
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = P[j], out[a.n + j] = H[j];
}

// The state at a segment's edge: h0 (or dh_end) through the segments before it (behind it).  Each wave composes a run
// of them, and the runs meet in LDS.  s: [kGsW][2][64 * V].
template <int V, bool MASK, bool BWD>
__device__ __forceinline__ void gs_enter(const GsArgs& a, int seg, int64_t c, const float* first, float (&h)[V],
                                         float (*s)[2][64 * V]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int W = blockDim.x >> 6;
#pragma unroll
  for (int j = 0; j < V; ++j) h[j] = first ? first[c + j] : 0.0f;
  const int count = BWD ? a.S - 1 - seg : seg;
  if (count == 0) return;  // for the whole workgroup
  const int per = (count + W - 1) / W, k0 = min(wave * per, count), k1 = min(k0 + per, count);
  float P[V], H[V];
#pragma unroll
  for (int j = 0; j < V; ++j) P[j] = 1.0f, H[j] = 0.0f;
#pragma unroll 4
  for (int k = k0; k < k1; ++k) {
    const float* m = a.part + (int64_t)(BWD ? a.S - 1 - k : k) * 2 * a.n + c;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      H[j] = gs_apply<MASK>(m[j], m[a.n + j], H[j]);
      P[j] = gs_product<MASK>(P[j], m[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) s[wave][0][lane * V + j] = P[j], s[wave][1][lane * V + j] = H[j];
  __syncthreads();
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = gs_apply<MASK>(s[w][0][lane * V + j], s[w][1][lane * V + j], h[j]);
  __syncthreads();
}

template <class T, int V, bool MASK>
__global__ __launch_bounds__(kGsW * 64) void k_gated(GsArgs a) {
  __shared__ float s_map[2][kGsW][2][64 * V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
  const int group = blockIdx.x % a.groups, seg = blockIdx.x / a.groups;
  const GsLane<T, V> at(a, group);
  const T *x = (const T*)a.x + at.x_at, *g = (const T*)a.g + at.g_at;
  T* out = (T*)a.h + at.c;
  const int64_t t0 = seg * a.len, t1 = min(a.T, t0 + a.len);
  float h[V];  // before the round
  gs_enter<V, MASK, false>(a, seg, at.c, a.h0, h, s_map[0]);
  GsRows<T, V> rx, rg;
  GsStarts rs;
  int64_t t = t0 + wave * kGsR;
  if (t < t1) {
    rx.load(x, a.x_st, t, t1), rg.load(g, a.g_st, t, t1);
    if (MASK) rs.load(a, at.b, t, t1);
  }
  int buf = 0;
  for (int64_t r = t0; r < t1; r += W * kGsR, t += W * kGsR, buf ^= 1) {
    float f[kGsR][V], b[kGsR][V], P[V], H[V];
#pragma unroll
    for (int j = 0; j < V; ++j) P[j] = 1.0f, H[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < kGsR; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float w;
        gs_gate(a.sigmoid, to_f(rg.v[i].v[j]), f[i][j], w);
        const float v = to_f(rx.v[i].v[j]);
        b[i][j] = a.mix ? w * v : v;
        if (MASK && rs.v[i]) f[i][j] = __builtin_bit_cast(float, kGsStart);
        if (t + i >= t1) f[i][j] = 1.0f, b[i][j] = 0.0f;
        H[j] = gs_apply<MASK>(f[i][j], b[i][j], H[j]);
        P[j] = gs_product<MASK>(P[j], f[i][j]);
      }
    if (const int64_t next = t + W * kGsR; next < t1) {
      rx.load(x, a.x_st, next, t1), rg.load(g, a.g_st, next, t1);
      if (MASK) rs.load(a, at.b, next, t1);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) s_map[buf][wave][0][lane * V + j] = P[j], s_map[buf][wave][1][lane * V + j] = H[j];
    __syncthreads();
    if (a.saved && wave == 0 && at.there)
#pragma unroll
      for (int j = 0; j < V; ++j) a.saved[r / kGsRows * a.n + at.c + j] = h[j];
    float mine[V];
#pragma unroll
    for (int j = 0; j < V; ++j) mine[j] = h[j];
    for (int w = 0; w < W; ++w) {
      if (w == wave)
#pragma unroll
        for (int j = 0; j < V; ++j) mine[j] = h[j];
#pragma unroll
      for (int j = 0; j < V; ++j)
        h[j] = gs_apply<MASK>(s_map[buf][w][0][lane * V + j], s_map[buf][w][1][lane * V + j], h[j]);
    }
#pragma unroll
    for (int i = 0; i < kGsR; ++i) {
      Vec<T, V> y;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        mine[j] = gs_apply<MASK>(f[i][j], b[i][j], mine[j]);
        y.v[j] = from_f<T>(mine[j]);
      }
      if (at.there && t + i < t1) *(Vec<T, V>*)(out + (t + i) * a.n) = y;
    }
  }
  if (t1 == a.T && wave == 0 && at.there)
#pragma unroll
    for (int j = 0; j < V; ++j) a.h_end[at.c + j] = h[j];
}

template <class T, int V, bool MASK>
__global__ __launch_bounds__(kGsW * 64) void k_gated_bwd(GsArgs a) {
  __shared__ float s_map[2][kGsW][3][64 * V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
  const int group = blockIdx.x % a.groups, seg = blockIdx.x / a.groups;
  const GsLane<T, V> at(a, group);
  const T *x = (const T*)a.x + at.x_at, *g = (const T*)a.g + at.g_at, *d = (const T*)a.dh + at.d_at;
  T *dx = (T*)a.dx + at.c, *dg = (T*)a.dg + at.c;
  const int64_t t0 = seg * a.len, t1 = min(a.T, t0 + a.len), rows = W * kGsR;
  float F[V];  // behind the round
  gs_enter<V, MASK, true>(a, seg, at.c, a.d_end, F, (float(*)[2][64 * V])s_map[0]);
  int buf = 0;
  for (int64_t r = t0 + (t1 - t0 - 1) / rows * rows; r >= t0 && t1 > t0; r -= rows, buf ^= 1) {
    const int64_t t = r + wave * kGsR;
    GsRows<T, V> rx, rg, rd;
    GsStarts rs;
    if (t < t1) {
      rx.load(x, a.x_st, t, t1), rg.load(g, a.g_st, t, t1);
      if (a.dh) rd.load(d, a.d_st, t, t1);
      if (MASK) rs.load(a, at.b, t, t1);
    }
    float h[V];  // before the round
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = a.saved[r / kGsRows * a.n + at.c + j];
    float f[kGsR][V], hp[kGsR][V], P[V], H[V], Q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) P[j] = 1.0f, H[j] = Q[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < kGsR; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float w;
        gs_gate(a.sigmoid, to_f(rg.v[i].v[j]), f[i][j], w);
        const float v = to_f(rx.v[i].v[j]);
        hp[i][j] = a.mix ? w * v : v;  // the row's input, until its state stands here
        if (MASK && rs.v[i]) f[i][j] = __builtin_bit_cast(float, kGsStart);
        if (t + i >= t1) f[i][j] = 1.0f, hp[i][j] = 0.0f;
        H[j] = gs_apply<MASK>(f[i][j], hp[i][j], H[j]);
        P[j] = gs_product<MASK>(P[j], f[i][j]);
      }
    auto grad = [&](int i, int j) { return a.dh && t + i < t1 ? to_f(rd.v[i].v[j]) : 0.0f; };
#pragma unroll
    for (int i = kGsR - 1; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        Q[j] = MASK && gs_marked(f[i][j]) ? 0.0f : f[i][j] * (grad(i, j) + Q[j]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s_map[buf][wave][0][lane * V + j] = P[j];
      s_map[buf][wave][1][lane * V + j] = H[j];
      s_map[buf][wave][2][lane * V + j] = Q[j];
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w)
#pragma unroll
      for (int j = 0; j < V; ++j)
        h[j] = gs_apply<MASK>(s_map[buf][w][0][lane * V + j], s_map[buf][w][1][lane * V + j], h[j]);
    float mine[V];
    for (int w = W - 1; w >= 0; --w) {
      if (w == wave)
#pragma unroll
        for (int j = 0; j < V; ++j) mine[j] = F[j];
#pragma unroll
      for (int j = 0; j < V; ++j)
        F[j] = gs_apply<MASK>(s_map[buf][w][0][lane * V + j], s_map[buf][w][2][lane * V + j], F[j]);
    }
#pragma unroll
    for (int i = 0; i < kGsR; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float b = hp[i][j];
        hp[i][j] = MASK && gs_marked(f[i][j]) ? 0.0f : h[j];
        h[j] = gs_apply<MASK>(f[i][j], b, h[j]);
      }
#pragma unroll
    for (int i = kGsR - 1; i >= 0; --i) {
      Vec<T, V> yx, yg;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float gate = to_f(rg.v[i].v[j]), v = to_f(rx.v[i].v[j]), E = grad(i, j) + mine[j];
        float p, w;
        gs_gate(a.sigmoid, gate, p, w);
        const float slope = a.sigmoid ? p * w : gate > 0.0f ? 0.0f : p;
        yx.v[j] = from_f<T>(a.mix ? w * E : E);
        yg.v[j] = from_f<T>(E * (a.mix ? hp[i][j] - v : hp[i][j]) * slope);
        mine[j] = MASK && gs_marked(f[i][j]) ? 0.0f : f[i][j] * E;
      }
      if (at.there && t + i < t1) {
        *(Vec<T, V>*)(dx + (t + i) * a.n) = yx;
        *(Vec<T, V>*)(dg + (t + i) * a.n) = yg;
      }
    }
  }
  if (a.dh0 && seg == 0 && wave == 0 && at.there)
#pragma unroll
    for (int j = 0; j < V; ++j) a.dh0[at.c + j] = F[j];
}

// One token: the state in place.
constexpr int kGsStep = 256;
template <class T, int V>
__global__ __launch_bounds__(kGsStep) void k_gated_step(GsArgs a, float* __restrict__ state) {
  const int64_t p = (int64_t)blockIdx.x * kGsStep + threadIdx.x;
  if (p >= a.pieces) return;
  const int64_t c = p * V, b = c / a.D, d = c - b * a.D;
  const Vec<T, V> x = *(const Vec<T, V>*)((const T*)a.x + b * a.x_sb + d);
  const Vec<T, V> g = *(const Vec<T, V>*)((const T*)a.g + b * a.g_sb + d);
  Vec<float, V> s = *(const Vec<float, V>*)(state + c);
  Vec<T, V> y;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float f, w;
    gs_gate(a.sigmoid, to_f(g.v[j]), f, w);
    const float v = to_f(x.v[j]);
    s.v[j] = __builtin_fmaf(f, s.v[j], a.mix ? w * v : v);
    y.v[j] = from_f<T>(s.v[j]);
  }
  *(Vec<float, V>*)(state + c) = s;
  *(Vec<T, V>*)((T*)a.h + c) = y;
}

static int gs_check(const lsh_gated* a) {
  if (!a || !lm_dtype_ok(a->dtype) || (a->decay != LSH_DECAY_SIGMOID && a->decay != LSH_DECAY_LOG)) return LSH_ERR_ARG;
  if (a->T < 0 || a->B < 0 || a->D < 1 || a->T > ((int64_t)1 << 40) || a->B > ((int64_t)1 << 40) ||
      a->D > ((int64_t)1 << 31) || (a->B > 0 && a->D > ((int64_t)1 << 40) / a->B) ||
      (a->T > 0 && a->B * a->D > ((int64_t)1 << 44) / a->T))
    return LSH_ERR_SHAPE;
  if (a->T > 0 && a->B > 0 && (bad_ptr(a->x) || bad_ptr(a->gate))) return LSH_ERR_ARG;
  return LSH_OK;
}

// Segments: as many as give the chip 512 workgroups (two a CU), of whole rounds; one where the channels alone give
// 384.  Returns the rows of a segment.
static int64_t gs_len(int64_t T, int64_t groups, int* S) {
  const int64_t rounds = (T + kGsRows - 1) / kGsRows;
  int64_t s = groups >= 384 ? 1 : (512 + groups - 1) / groups;
  if (s > rounds) s = rounds;
  if (s < 1) s = 1;
  const int64_t per = (rounds + s - 1) / s;
  *S = (int)(per ? (rounds + per - 1) / per : 1);
  return per * kGsRows;
}
static int64_t gs_groups(const lsh_gated* a, int V) { return (a->B * a->D + 64 * V - 1) / (64 * V); }

static GsArgs gs_args(const lsh_gated* p) {
  GsArgs a = {};
  a.x = p->x, a.g = p->gate, a.x_st = p->x_st, a.x_sb = p->x_sb, a.g_st = p->g_st, a.g_sb = p->g_sb;
  a.starts = p->starts, a.h0 = p->h0;
  a.T = p->T, a.B = p->B, a.D = p->D, a.n = p->B * p->D;
  a.sigmoid = p->decay == LSH_DECAY_SIGMOID, a.mix = p->mix != 0;
  return a;
}
// Whether pieces of V elements can be read at once: their addresses are multiples of their size.
static bool gs_wide(const GsArgs& a, int size, int V) {
  if (a.D % V) return false;
  const int bytes = size * V;
  for (const void* p : {a.x, a.g, a.dh, (const void*)a.h, (const void*)a.dx, (const void*)a.dg})
    if ((uintptr_t)p % bytes) return false;
  for (int64_t s : {a.x_st, a.x_sb, a.g_st, a.g_sb, a.d_st, a.d_sb})
    if (s % V) return false;
  return true;
}
template <class F>
static void with_mask(bool mask, F&& f) {
  if (mask)
    f(std::true_type{});
  else
    f(std::false_type{});
}
static size_t gs_workspace(const lsh_gated* p) {
  size_t most = 0;
  if (p->B == 0) return 0;
  for (int V : {1, 2}) {
    int S;
    gs_len(p->T, gs_groups(p, V), &S);
    if (S > 1) most = std::max(most, (size_t)S * 2 * p->B * p->D * sizeof(float));
  }
  return most;
}

// Calls f<T, V, MASK>(threads of a workgroup, workgroups), everything about the launch in *a.  False: too many.
template <class F>
static bool gs_launch(GsArgs& a, int dtype, F&& f) {
  const bool two = gs_wide(a, lm_dtype_size(dtype), 2);
  a.pieces = a.n / (two ? 2 : 1);
  const int64_t groups = (a.pieces + 63) / 64;
  a.len = gs_len(a.T, groups, &a.S);
  if (!lm_grid_ok(groups * a.S, kGsW * 64)) return false;
  a.groups = (int)groups;
  // of short sequences as many waves as there are rows for
  const int W = a.T > kGsRows / 2 ? kGsW : a.T > kGsRows / 4 ? kGsW / 2 : a.T > kGsR ? kGsW / 4 : 1;
  with_dtype(dtype, [&](auto t) {
    with_mask(a.starts != nullptr, [&](auto mask) {
      if (two)
        f(t, std::integral_constant<int, 2>{}, mask, W * 64, (unsigned)(groups * a.S));
      else
        f(t, std::integral_constant<int, 1>{}, mask, W * 64, (unsigned)(groups * a.S));
    });
  });
  return true;
}

}  // namespace lsh

using namespace lsh;

extern "C" int64_t lsh_gated_saved(const lsh_gated* p) {
  if (gs_check(p)) return 0;
  return (p->T + kGsRows - 1) / kGsRows * p->B * p->D;
}

extern "C" size_t lsh_gated_workspace(const lsh_gated* p) { return gs_check(p) ? 0 : gs_workspace(p); }

extern "C" int lsh_gated_fwd(const lsh_gated* p, void* h, float* h_end, float* saved, void* ws, size_t ws_bytes,
                             void* stream) {
  if (int rc = gs_check(p)) return rc;
  if (p->B == 0) return LSH_OK;
  if ((p->T > 0 && bad_ptr(h)) || bad_ptr(h_end)) return LSH_ERR_ARG;
  const size_t need = gs_workspace(p);
  if (need && (bad_ptr(ws) || ws_bytes < need)) return LSH_ERR_WORKSPACE;
  GsArgs a = gs_args(p);
  a.h = h, a.h_end = h_end, a.saved = saved, a.part = (float*)ws;
  hipStream_t st = (hipStream_t)stream;
  if (!gs_launch(a, p->dtype, [&](auto t, auto v, auto mask, int threads, unsigned grid) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        constexpr bool MASK = decltype(mask)::value;
        if (a.S > 1) k_gated_sums<T, V, MASK, false><<<dim3(grid), kGsW * 64, 0, st>>>(a);
        k_gated<T, V, MASK><<<dim3(grid), threads, 0, st>>>(a);
      }))
    return LSH_ERR_SHAPE;
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" int lsh_gated_bwd(const lsh_gated* p, const float* saved, const void* dh, int64_t dh_st, int64_t dh_sb,
                             const float* dh_end, void* dx, void* dgate, float* dh0, void* ws, size_t ws_bytes,
                             void* stream) {
  if (int rc = gs_check(p)) return rc;
  if (p->B == 0) return LSH_OK;
  if (p->T > 0 && (bad_ptr(saved) || bad_ptr(dx) || bad_ptr(dgate))) return LSH_ERR_ARG;
  const size_t need = gs_workspace(p);
  if (need && (bad_ptr(ws) || ws_bytes < need)) return LSH_ERR_WORKSPACE;
  GsArgs a = gs_args(p);
  a.saved = (float*)saved, a.dh = dh, a.d_st = dh ? dh_st : 0, a.d_sb = dh ? dh_sb : 0, a.d_end = dh_end;
  a.dx = dx, a.dg = dgate, a.dh0 = dh0, a.part = (float*)ws;
  hipStream_t st = (hipStream_t)stream;
  if (!gs_launch(a, p->dtype, [&](auto t, auto v, auto mask, int threads, unsigned grid) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        constexpr bool MASK = decltype(mask)::value;
        if (a.S > 1) k_gated_sums<T, V, MASK, true><<<dim3(grid), kGsW * 64, 0, st>>>(a);
        k_gated_bwd<T, V, MASK><<<dim3(grid), threads, 0, st>>>(a);
      }))
    return LSH_ERR_SHAPE;
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" int lsh_gated_step(const lsh_gated* p, float* state, void* h, void* stream) {
  if (int rc = gs_check(p)) return rc;
  if (p->T != 1) return LSH_ERR_SHAPE;
  if (p->B == 0) return LSH_OK;
  if (bad_ptr(state) || bad_ptr(h)) return LSH_ERR_ARG;
  GsArgs a = gs_args(p);
  a.h = h, a.x_st = a.g_st = 0;
  const bool four = gs_wide(a, lm_dtype_size(p->dtype), 4) && (uintptr_t)state % 16 == 0;
  a.pieces = a.n / (four ? 4 : 1);
  const int64_t groups = (a.pieces + kGsStep - 1) / kGsStep;
  if (!lm_grid_ok(groups, kGsStep)) return LSH_ERR_SHAPE;
  with_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    if (four)
      k_gated_step<T, 4><<<dim3((unsigned)groups), kGsStep, 0, (hipStream_t)stream>>>(a, state);
    else
      k_gated_step<T, 1><<<dim3((unsigned)groups), kGsStep, 0, (hipStream_t)stream>>>(a, state);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
