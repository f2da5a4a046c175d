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
// F_begin = P*F_end + Q and the same P.  A lane has V neighbouring channels, a wave 8 rows of them in registers,
// and a workgroup's waves hold consecutive rows: the waves' maps meet in LDS, each wave composes those before its own,
// and then writes its rows from the state before them.  Where there are too few channels for the chip the rows are cut
// into segments, whose maps an extra pass over the operands forms.  The gradients take h_{t-1} from the state before
// every kGsSave rows, which the forward keeps in fp32, and form it again: h itself may have 16 bits.
//
// A start is a factor -0 (decays are never negative): a marked product stays marked and drops what it is
// applied to, also an infinity or a NaN.
#include <algorithm>
#include <type_traits>

#include "lsh_lm.h"

namespace lsh {

// Waves of a workgroup, what the rows of a segment are a multiple of, and the rows between saved states.
constexpr int kGsW = 8, kGsRows = 128, kGsSave = 64;
// Rows that a wave holds: forwards, backwards, and for a segment's map with so many bytes a lane and row.  (16 rows
// forwards have not the registers for two workgroups a CU in every type: fp16 4096 x 4 x 2048 57 us, so 40; bf16 41, so 39.)
constexpr int kGsFwd = 8, kGsBwd = 8;
template <int BYTES>
constexpr int kGsSum = BYTES == 8 ? 8 : 16;

struct GsArgs {
  const void *x, *g;
  int64_t x_st, x_sb, g_st, g_sb;
  const uint8_t* starts;  // [T, B], or NULL
  const float* h0;        // [n], or NULL
  void* h;
  float *h_end, *saved;   // saved: the states before every kGsSave rows, or NULL
  const void* dh;
  int64_t d_st, d_sb;
  const float* d_end;
  void *dx, *dg;
  float* dh0;
  float* part;            // [S, 2, n]: the segments' maps
  int64_t T, B, D, n, pieces, len;  // n = B*D channels in pieces of V; rows of a segment
  int groups, S, sigmoid, mix;
};

// e^x for x <= 0: the hardware's power of two with what the product x*log2(e) loses put back.  16-bit gates go without
// (6 instructions of 30 an element): it is |x|*2^-24 of a decay.  What is rounded to 16 bits does not show it, and the
// states and dh0, which are fp32, hardly (1024 rows of 4096 channels, of the states' norm: sigmoid bf16 0.97e-7, with it
// 0.94e-7, fp16 1.00e-7 and 0.95e-7; log decays 0.78e-7 and 0.80e-7 either way; dh0 over 64 rows 2.0e-7 to 2.2e-7 either way).
template <bool FINE>
__device__ __forceinline__ float gs_exp(float x) {
  constexpr float kHi = 1.44269502f, kLo = 1.92596299e-8f;  // log2(e)
  if constexpr (!FINE) return __builtin_amdgcn_exp2f(x * kHi);
  x = x < -150.0f ? -150.0f : x;  // 0, and no inf - inf; a NaN stays
  const float t = x * kHi, r = __builtin_fmaf(x, kHi, -t) + x * kLo;
  const float y = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(y, r * 0.693147181f, y);
}

// (a, 1 - a).  Of a sigmoid the smaller one is e/(1 + e) with e = exp(-|g|), 1 - e^g is a Taylor sum where it would
// cancel, and a decay near one is what is left of one: it is raised to hundreds of rows, so it is rounded once (with
// the hardware's 1/(1 + e) and 2^x in its place the results of 1000 rows in fp32 were off by 7.2e-7 of their norm, so 2.2e-7).
template <bool FINE, bool SIGMOID>
__device__ __forceinline__ void gs_gate(float g, float& a, float& w) {
  if constexpr (SIGMOID) {
    const float e = gs_exp<FINE>(-__builtin_fabsf(g)), s = e * __builtin_amdgcn_rcpf(1.0f + e), r = 1.0f - s;
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
    const float e = gs_exp<FINE>(g);
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

// Bytes of a lane in a row: 8, 4, or one element of either size.  The first two have a row's lanes within 4 GB of each
// other, so that an address is a scalar and an offset; the last reads a channel wherever it lies.  Wider is faster for
// the maps (4096 x 4 x 2048 bf16: 36 us with 8 bytes, 41 with 4, 54 with 2), but the passes themselves have not the
// registers for 8 (forward 61 us with 8 rows a wave of 8 bytes, 39 with 8 rows of 4, 55 with 16 rows of 2).
template <class T, int BYTES>
constexpr int kGsV = BYTES > (int)sizeof(T) ? BYTES / (int)sizeof(T) : 1;
template <int BYTES>
using GsOff = std::conditional_t<BYTES != 0, uint32_t, uint64_t>;

// A lane's channels.  A lane beyond the last channel does the last ones once more, to the same values.
template <class T, int BYTES>
struct GsLane {
  static constexpr int V = kGsV<T, BYTES>;
  int64_t c0, c, b0, b, d;  // the first channel of the wave and of the lane, their batches, the lane's column
  __device__ __forceinline__ GsLane(const GsArgs& a, int group) {
    const int64_t p0 = (int64_t)group * 64, p = min(p0 + (threadIdx.x & 63), a.pieces - 1);
    c0 = p0 * V, c = p * V;
    b0 = c0 / a.D, b = c / a.D, d = c - b * a.D;
  }
};

// A lane's V values of a row as they lie in memory: two of 16 bits stay in one register.
template <class T, int V>
struct alignas(V * sizeof(T)) GsRaw {
  using Word = std::conditional_t<V * sizeof(T) >= 4, uint32_t, uint16_t>;
  static constexpr int N = V * sizeof(T) / sizeof(Word), PER = sizeof(Word) / sizeof(T);
  Word x[N];
  __device__ __forceinline__ float get(int j) const {
    const Word w = x[j / PER];
    if constexpr (PER == 1)
      return to_f(__builtin_bit_cast(T, w));
    else if constexpr (std::is_same_v<T, bf16_t>)
      return __builtin_bit_cast(float, j % 2 ? w & 0xffff0000u : w << 16);
    else
      return to_f(__builtin_bit_cast(T, (uint16_t)(w >> 16 * (j % 2))));
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
    Vec<T, V> y;
#pragma unroll
    for (int j = 0; j < V; ++j) y.v[j] = from_f<T>(f[j]);
    __builtin_memcpy(x, &y, sizeof(y));
  }
};

// One operand as a lane reads it, row by row
template <class T, int BYTES>
struct GsIn {
  static constexpr int V = kGsV<T, BYTES>;
  const T* base;
  int64_t stride;
  GsOff<BYTES> off;
  __device__ __forceinline__ GsIn(const void* p, int64_t st, int64_t sb, const GsLane<T, BYTES>& at)
      : base((const T*)p + at.b0 * sb), stride(st), off((GsOff<BYTES>)(((at.b - at.b0) * sb + at.d) * sizeof(T))) {}
  __device__ __forceinline__ GsRaw<T, V> row(int64_t t) const {
    return *(const GsRaw<T, V>*)((const char*)(base + t * stride) + off);
  }
};
template <class T, int BYTES>
struct GsOut {
  static constexpr int V = kGsV<T, BYTES>;
  T* base;
  int64_t n;
  uint32_t off;
  __device__ __forceinline__ GsOut(void* p, int64_t n, const GsLane<T, BYTES>& at)
      : base((T*)p + at.c0), n(n), off((uint32_t)((at.c - at.c0) * sizeof(T))) {}
  __device__ __forceinline__ void put(int64_t t, const float (&f)[V]) const {
    GsRaw<T, V> x;
    x.set(f);
    *(GsRaw<T, V>*)((char*)(base + t * n) + off) = x;
  }
};

// R rows of a lane as read; rows from `end` on are read from the one before it
template <class T, int BYTES, int R>
struct GsRows {
  GsRaw<T, kGsV<T, BYTES>> v[R];
  __device__ __forceinline__ void load(const GsIn<T, BYTES>& in, int64_t t, int64_t end) {
    if (t + R <= end) {
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] = in.row(t + i);
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] = in.row(t + i < end ? t + i : end - 1);
    }
  }
  __device__ __forceinline__ float get(int i, int j) const { return v[i].get(j); }
};
// A bit for each of R rows that starts a sequence
template <bool MASK, int R>
__device__ __forceinline__ unsigned gs_starts(const GsArgs& a, int64_t b, int64_t t, int64_t end) {
  unsigned bits = 0;
  if constexpr (MASK)
    if (t < end) {
      uint8_t v[R];
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] = a.starts[(t + i < end ? t + i : end - 1) * a.B + b];
#pragma unroll
      for (int i = 0; i < R; ++i) bits |= (v[i] != 0) << i;
    }
  return bits;
}
__device__ __forceinline__ bool gs_bit(unsigned bits, int i) { return bits >> i & 1; }

// Calls f with whether the decay is a sigmoid and whether inputs are weighed, as constants: the branch stands once
// around a chunk of rows.
template <class F>
__device__ __forceinline__ void gs_form(const GsArgs& a, F&& f) {
  if (a.sigmoid) {
    if (a.mix)
      f(std::true_type{}, std::true_type{});
    else
      f(std::true_type{}, std::false_type{});
  } else {
    if (a.mix)
      f(std::false_type{}, std::true_type{});
    else
      f(std::false_type{}, std::false_type{});
  }
}

// Where segments are needed: the map of each but the last, forwards (x, gate), or of each but the first, backwards
// (gate, dh).  A wave takes its share of the segment's rows, its map in registers; backwards the map is summed with
// the product of the decays so far, from the first row on.
template <int BYTES>
constexpr int kGsSumW = BYTES == 8 ? 8 : 4;
template <class T, int BYTES, bool MASK, bool BWD>
__global__ __launch_bounds__(kGsSumW<BYTES> * 64, 4) void k_gated_sums(GsArgs a) {
  constexpr int V = kGsV<T, BYTES>, R = kGsSum<BYTES>;
  __shared__ float s_map[kGsSumW<BYTES>][2][64 * V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = blockIdx.x % a.groups, seg = blockIdx.x / a.groups + (BWD ? 1 : 0);
  const GsLane<T, BYTES> at(a, group);
  const GsIn<T, BYTES> x = BWD ? GsIn<T, BYTES>(a.dh, a.d_st, a.d_sb, at) : GsIn<T, BYTES>(a.x, a.x_st, a.x_sb, at);
  const GsIn<T, BYTES> g(a.g, a.g_st, a.g_sb, at);
  const int64_t t1 = min(a.T, (seg + 1) * a.len);
  const int64_t per = a.len / kGsSumW<BYTES>, lo = seg * a.len + wave * per, hi = min(t1, lo + per);
  float P[V], H[V];
#pragma unroll
  for (int j = 0; j < V; ++j) P[j] = 1.0f, H[j] = 0.0f;
  const bool zeros = BWD && !a.dh;
  GsRows<T, BYTES, R> nx, ng;
  auto load = [&](int64_t t) {
    if (!zeros) nx.load(x, t, hi);
    ng.load(g, t, hi);
  };
  if (lo < hi) load(lo);
  for (int64_t t = lo; t < hi; t += R) {
    const GsRows<T, BYTES, R> rx = nx, rg = ng;
    const unsigned starts = gs_starts<MASK, R>(a, at.b, t, hi);
    if (t + R < hi) load(t + R);
    gs_form(a, [&](auto sig, auto mix) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (t + i >= hi) break;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float f, w;
          gs_gate<sizeof(T) == 4, decltype(sig)::value>(rg.get(i, j), f, w);
          if (MASK && gs_bit(starts, i)) f = __builtin_bit_cast(float, kGsStart);
          P[j] = gs_product<MASK>(P[j], f);
          const float v = BWD && zeros ? 0.0f : rx.get(i, j);
          if constexpr (BWD)
            H[j] = MASK && gs_marked(P[j]) ? H[j] : __builtin_fmaf(P[j], v, H[j]);
          else
            H[j] = gs_apply<MASK>(f, decltype(mix)::value ? w * v : v, H[j]);
        }
      }
    });
  }
#pragma unroll
  for (int j = 0; j < V; ++j) s_map[wave][0][lane * V + j] = P[j], s_map[wave][1][lane * V + j] = H[j];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int j = 0; j < V; ++j) P[j] = 1.0f, H[j] = 0.0f;
#pragma unroll
  for (int n = 0; n < kGsSumW<BYTES>; ++n) {
    const int w = BWD ? kGsSumW<BYTES> - 1 - n : n;
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

// One barrier a round: what a wave writes for the next round goes to the other half of the LDS.  The state after a
// round is what its last wave ends with.
template <class T, int BYTES, bool MASK>
__global__ __launch_bounds__(kGsW * 64, 4) void k_gated(GsArgs a) {
  constexpr int V = kGsV<T, BYTES>, R = kGsFwd;
  __shared__ float s_map[2][kGsW][2][64 * V], s_carry[2][64 * V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
  const int group = blockIdx.x % a.groups, seg = blockIdx.x / a.groups;
  const GsLane<T, BYTES> at(a, group);
  const GsIn<T, BYTES> x(a.x, a.x_st, a.x_sb, at), g(a.g, a.g_st, a.g_sb, at);
  const GsOut<T, BYTES> out(a.h, a.n, at);
  const int64_t t0 = seg * a.len, t1 = min(a.T, t0 + a.len);
  GsRows<T, BYTES, R> rx, rg;
  int64_t t = t0 + wave * R;
  auto load = [&](int64_t t) { rx.load(x, t, t1), rg.load(g, t, t1); };
  if (t < t1) load(t);
  float h[V];  // before the round, then before the wave's rows
  gs_enter<V, MASK, false>(a, seg, at.c, a.h0, h, s_map[0]);
  if (wave == W - 1)
#pragma unroll
    for (int j = 0; j < V; ++j) s_carry[0][lane * V + j] = h[j];
  int buf = 0;
  for (int64_t r = t0; r < t1; r += W * R, t += W * R, buf ^= 1) {
    float f[R][V], b[R][V], P[V], H[V];
    const unsigned starts = gs_starts<MASK, R>(a, at.b, t, t1);
    gs_form(a, [&](auto sig, auto mix) {
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float w;
          gs_gate<sizeof(T) == 4, decltype(sig)::value>(rg.get(i, j), f[i][j], w);
          b[i][j] = decltype(mix)::value ? w * rx.get(i, j) : rx.get(i, j);
        }
    });
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (MASK && gs_bit(starts, i)) f[i][j] = __builtin_bit_cast(float, kGsStart);
    if (t + R > t1)
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (t + i >= t1)
#pragma unroll
          for (int j = 0; j < V; ++j) f[i][j] = 1.0f, b[i][j] = 0.0f;
    if (const int64_t next = t + W * R; next < t1) load(next);
#pragma unroll
    for (int j = 0; j < V; ++j) P[j] = 1.0f, H[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        H[j] = gs_apply<MASK>(f[i][j], b[i][j], H[j]);
        P[j] = gs_product<MASK>(P[j], f[i][j]);
      }
#pragma unroll
    for (int j = 0; j < V; ++j) s_map[buf][wave][0][lane * V + j] = P[j], s_map[buf][wave][1][lane * V + j] = H[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = s_carry[buf][lane * V + j];
    for (int w = 0; w < wave; ++w)
#pragma unroll
      for (int j = 0; j < V; ++j)
        h[j] = gs_apply<MASK>(s_map[buf][w][0][lane * V + j], s_map[buf][w][1][lane * V + j], h[j]);
    if (a.saved && t % kGsSave == 0 && t < t1)
#pragma unroll
      for (int j = 0; j < V; ++j) a.saved[t / kGsSave * a.n + at.c + j] = h[j];
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) h[j] = gs_apply<MASK>(f[i][j], b[i][j], h[j]);
      if (t + i < t1) out.put(t + i, h);
    }
    if (wave == W - 1)
#pragma unroll
      for (int j = 0; j < V; ++j) s_carry[buf ^ 1][lane * V + j] = h[j];
  }
  if (t1 == a.T && wave == W - 1)
#pragma unroll
    for (int j = 0; j < V; ++j) a.h_end[at.c + j] = h[j];
}

// The gradients, the rounds from the last.  A first sweep over the rows in registers forms the wave's maps of both
// directions, a second one forwards the states and what multiplies the adjoint, a third one backwards the adjoint: the
// gates' powers are formed twice, which is cheaper than keeping them (two workgroups a CU need 128 registers).
template <class T, int BYTES, bool MASK>
__global__ __launch_bounds__(kGsW * 64, 4) void k_gated_bwd(GsArgs a) {
  constexpr int V = kGsV<T, BYTES>, R = kGsBwd;
  __shared__ float s_map[2][kGsW][3][64 * V], s_carry[2][64 * V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
  const int group = blockIdx.x % a.groups, seg = blockIdx.x / a.groups;
  const GsLane<T, BYTES> at(a, group);
  const GsIn<T, BYTES> x(a.x, a.x_st, a.x_sb, at), g(a.g, a.g_st, a.g_sb, at), d(a.dh, a.d_st, a.d_sb, at);
  const GsOut<T, BYTES> dx(a.dx, a.n, at), dg(a.dg, a.n, at);
  const int64_t t0 = seg * a.len, t1 = min(a.T, t0 + a.len), rows = W * R;
  float F[V];  // behind the round, then behind the wave's rows
  gs_enter<V, MASK, true>(a, seg, at.c, a.d_end, F, (float(*)[2][64 * V])s_map[0]);
  if (wave == 0)
#pragma unroll
    for (int j = 0; j < V; ++j) s_carry[0][lane * V + j] = F[j];
  int buf = 0;
  for (int64_t r = t0 + (t1 - t0 - 1) / rows * rows; r >= t0 && t1 > t0; r -= rows, buf ^= 1) {
    const int64_t t = r + wave * R;
    GsRows<T, BYTES, R> rx, rg, rd;
    if (t < t1) {
      rx.load(x, t, t1), rg.load(g, t, t1);
      if (a.dh) rd.load(d, t, t1);
    }
    const unsigned starts = gs_starts<MASK, R>(a, at.b, t, t1);
    float h[V];  // before the round, then before the wave's rows
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = a.saved[r / kGsSave * a.n + at.c + j];
    // rows that are not there: a decay of 1, an input and a gradient of 0
    const bool tail = t + R > t1;
    if (tail || !a.dh)
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (t + i >= t1 || !a.dh)
#pragma unroll
          for (auto& word : rd.v[i].x) word = 0;
    float P[V], H[V], Q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) P[j] = 1.0f, H[j] = Q[j] = 0.0f;
    gs_form(a, [&](auto sig, auto mix) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (tail && t + i >= t1) break;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float f, w;
          gs_gate<sizeof(T) == 4, decltype(sig)::value>(rg.get(i, j), f, w);
          if (MASK && gs_bit(starts, i)) f = __builtin_bit_cast(float, kGsStart);
          H[j] = gs_apply<MASK>(f, decltype(mix)::value ? w * rx.get(i, j) : rx.get(i, j), H[j]);
          P[j] = gs_product<MASK>(P[j], f);
          Q[j] = MASK && gs_marked(P[j]) ? Q[j] : __builtin_fmaf(P[j], rd.get(i, j), Q[j]);
        }
      }
    });
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
#pragma unroll
    for (int j = 0; j < V; ++j) F[j] = s_carry[buf][lane * V + j];
    for (int w = W - 1; w > wave; --w)
#pragma unroll
      for (int j = 0; j < V; ++j)
        F[j] = gs_apply<MASK>(s_map[buf][w][0][lane * V + j], s_map[buf][w][2][lane * V + j], F[j]);
    // the first sweep's values are not to be kept for the second
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int k = 0; k < GsRaw<T, V>::N; ++k) asm volatile("" : "+v"(rg.v[i].x[k]), "+v"(rx.v[i].x[k]));
    // dx = w*E, dgate = u*E, F = f*E
    float f[R][V], w[R][V], u[R][V];
    gs_form(a, [&](auto sig, auto mix) {
      constexpr bool SIG = decltype(sig)::value, MIX = decltype(mix)::value;
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float gate = rg.get(i, j), v = rx.get(i, j);
          float p, q;
          gs_gate<sizeof(T) == 4, SIG>(gate, p, q);
          const float slope = SIG ? p * q : gate > 0.0f ? 0.0f : p;
          const bool start = MASK && gs_bit(starts, i);
          const float before = start ? 0.0f : h[j];
          u[i][j] = (MIX ? before - v : before) * slope;
          w[i][j] = MIX ? q : 1.0f;
          f[i][j] = start ? __builtin_bit_cast(float, kGsStart) : p;
          h[j] = __builtin_fmaf(p, before, MIX ? q * v : v);
        }
    });
    if (tail)
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (t + i >= t1)
#pragma unroll
          for (int j = 0; j < V; ++j) f[i][j] = 1.0f;
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      float yx[V], yg[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float E = rd.get(i, j) + F[j];
        yx[j] = w[i][j] * E;
        yg[j] = u[i][j] * E;
        F[j] = MASK && gs_marked(f[i][j]) ? 0.0f : f[i][j] * E;
      }
      if (t + i < t1) dx.put(t + i, yx), dg.put(t + i, yg);
    }
    if (wave == 0)
#pragma unroll
      for (int j = 0; j < V; ++j) s_carry[buf ^ 1][lane * V + j] = F[j];
  }
  if (a.dh0 && seg == 0 && wave == 0)
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
    if (a.sigmoid)
      gs_gate<sizeof(T) == 4, true>(to_f(g.v[j]), f, w);
    else
      gs_gate<sizeof(T) == 4, false>(to_f(g.v[j]), f, w);
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
// 384.  Returns the rows of a segment.  (4096 x 4 x 2048 bf16 with 256 workgroups: forward 43 us, gradients 91, so 39 and
// 75; with 768 the maps take 45, so 36.)
static int64_t gs_len(int64_t T, int64_t groups, int* S) {
  const int64_t rounds = (T + kGsRows - 1) / kGsRows;
  int64_t s = groups >= 384 ? 1 : (512 + groups - 1) / groups;
  if (s > rounds) s = rounds;
  if (s < 1) s = 1;
  const int64_t per = (rounds + s - 1) / s;
  *S = (int)(per ? (rounds + per - 1) / per : 1);
  return per * kGsRows;
}

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
    gs_len(p->T, (p->B * p->D + 64 * V - 1) / (64 * V), &S);
    if (S > 1) most = std::max(most, (size_t)S * 2 * p->B * p->D * sizeof(float));
  }
  return most;
}

// Whether a wave's lanes lie within 32-bit offsets of each other in each operand: it may reach over several batches.
static bool gs_near(const GsArgs& a, int size, int V) {
  const int64_t over = std::min<int64_t>(a.B - 1, 64 * V / a.D + 1);
  for (int64_t sb : {a.x_sb, a.g_sb, a.d_sb})
    if (sb < 0 || (over > 0 && sb > (((int64_t)1 << 32) / size - a.D) / over)) return false;
  return a.D < ((int64_t)1 << 32) / size;
}

// Bytes of a lane in a row, at most `most`: 8 or 4 where all operands allow it, else 0 (one channel anywhere).
static int gs_bytes(const GsArgs& a, int size, int most) {
  for (int bytes = most; bytes >= 4; bytes /= 2)
    if (const int V = bytes / size; (V == 1 || gs_wide(a, size, V)) && gs_near(a, size, V)) return bytes;
  return 0;
}
template <class F>
static void with_bytes(int bytes, F&& f) {
  if (bytes == 8)
    f(std::integral_constant<int, 8>{});
  else if (bytes == 4)
    f(std::integral_constant<int, 4>{});
  else
    f(std::integral_constant<int, 0>{});
}
// The channels in groups of 64 pieces
static void gs_group(GsArgs& a, int size, int bytes) {
  a.pieces = a.n / (bytes ? bytes / size : 1);
  a.groups = (int)((a.pieces + 63) / 64);
}

template <bool BWD>
static int gs_run(GsArgs& a, int dtype, hipStream_t st) {
  const int size = lm_dtype_size(dtype);
  if (!lm_grid_ok(a.n / 64 + 1, kGsW * 64)) return LSH_ERR_SHAPE;
  const int bytes = gs_bytes(a, size, 4), sums = gs_bytes(a, size, 8);
  gs_group(a, size, bytes);
  a.len = gs_len(a.T, a.groups, &a.S);
  if (!lm_grid_ok((int64_t)a.groups * a.S, kGsW * 64)) return LSH_ERR_SHAPE;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    with_mask(a.starts != nullptr, [&](auto mask) {
      constexpr bool MASK = decltype(mask)::value;
      if (a.S > 1)
        with_bytes(sums, [&](auto n) {
          constexpr int N = decltype(n)::value;
          GsArgs b = a;
          gs_group(b, size, N);
          k_gated_sums<T, N, MASK, BWD><<<dim3(b.groups * (b.S - 1)), kGsSumW<N> * 64, 0, st>>>(b);
        });
      with_bytes(bytes, [&](auto n) {
        constexpr int N = decltype(n)::value;
        if constexpr (N <= 4) {
          constexpr int R = BWD ? kGsBwd : kGsFwd;
          // of short sequences as many waves as there are rows for
          const int W = a.T > 4 * R ? 8 : a.T > 2 * R ? 4 : a.T > R ? 2 : 1;
          if constexpr (BWD)
            k_gated_bwd<T, N, MASK><<<dim3(a.groups * a.S), W * 64, 0, st>>>(a);
          else
            k_gated<T, N, MASK><<<dim3(a.groups * a.S), W * 64, 0, st>>>(a);
        }
      });
    });
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

}  // namespace lsh

using namespace lsh;

extern "C" int64_t lsh_gated_saved(const lsh_gated* p) {
  if (gs_check(p)) return 0;
  return (p->T + kGsSave - 1) / kGsSave * p->B * p->D;
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
  return gs_run<false>(a, p->dtype, (hipStream_t)stream);
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
  return gs_run<true>(a, p->dtype, (hipStream_t)stream);
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
