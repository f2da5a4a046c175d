// The norm after a block, its gate and residual scale, and the norm before the next block, as one
// pass over the rows (and one for the gradients):
//
//   n = y * ry * w_post,  ry = 1/sqrt(mean(y^2) + eps)        the block's output, normalised
//   h = act(gate) * n                                         silu or sigmoid, or no gate
//   x_new = x + a*h                                           a: one number or one a channel
//   z = x_new * rx * w_pre,  rx = 1/sqrt(mean(x_new^2) + eps) the next block's input
//
// Gradients, with gx and gz those of x_new and z and <.> the mean over the row:
//   u = gz*w_pre,    dx = gx + rx*(u - x_new*rx^2*<u*x_new>)
//   dn = a*dx*act,   dgate = a*dx*n*act'(gate)
//   m = dn*w_post,   dy = ry*(m - y*ry^2*<m*y>)
//   dw_pre = sum gz*x_new*rx,  dw_post = sum dn*y*ry,  da = sum dx*h      over the rows
// Bound by the rows' bytes; x_new is computed again instead of being kept.  bf16, 8192 x 2048: forward
// 26.6 us for 168 MB (6.3 TB/s, part of it from the Infinity Cache), gradients 48 us for 268 MB
// (5.6 TB/s) and 4.4 for the parameters' sums; with an fp32 stream 35 and 75, all fp32 62 and 106.  Rows
// that cannot be read in pieces go element by element: 8190 x 2047 forward 28, gradients 63.
#include <type_traits>

#include "lsh_lm.h"

namespace lsh {

struct BnArgs {
  const void *x, *y, *gate;
  const float *w_post, *w_pre, *scale;  // scale: per channel, or NULL (scale1)
  float scale1, eps;
  int act;
  int64_t rows;
  int D;
  void *x_new, *z;
  const void *gx, *gz;
  void *dx, *dy, *dgate;
  float* part;  // [grid, 3, D]: this workgroup's sums of dw_post, dw_pre and da
};

// Sums over the lanes that share a row: one wave, or all W of the workgroup (through s).  The waves' sums
// are added as a tree over W neighbouring lanes, N reads a lane instead of N*W (those take up to 80
// registers).  One barrier: s is written again only after a barrier behind the next call's, which has
// another s.
template <int W, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* s) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum_f(v[i]);
  if constexpr (W > 1) {
    static_assert(W <= 16, "within a row of 16 lanes");
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[w * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = s[(threadIdx.x & (W - 1)) * N + i];
      if constexpr (W > 8) v[i] += row_turned<8>(v[i]);
      if constexpr (W > 4) v[i] += row_turned<4>(v[i]);
      if constexpr (W > 2) v[i] += row_turned<2>(v[i]);
      v[i] += row_turned<1>(v[i]);
    }
  }
}

// A row of D values (or of none) at a wave-uniform address.  Columns beyond it read as zeros and are not
// written, without branches or selects: the buffer's bounds do it.
template <class T>
struct BnRow {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ BnRow(const void* p, int64_t row, int D, bool there = true)
      : r(__builtin_amdgcn_make_buffer_rsrc((T*)const_cast<void*>(p) + (size_t)row * D, (short)0,
                                            there ? D * (int)sizeof(T) : 0, 0x00020000)) {}
};

using u32x2 = unsigned __attribute__((ext_vector_type(2)));
using u32x4 = unsigned __attribute__((ext_vector_type(4)));

// A lane's piece of V values, the d/V-th of the row.  WIDE: columns d.., in accesses of 8 or 16 bytes.
// Otherwise one by one, the columns dealt out so that a wave's lanes read neighbours (8190 x 2047 forward
// 28 us and gradients 63, with a lane's own columns side by side 128 and 106).
template <int V, bool WIDE>
__device__ __forceinline__ int bn_col(int d, int j) {
  return WIDE ? d + j : (d / V & ~63) * V + j * 64 + (d / V & 63);
}
template <int V, bool WIDE, class T>
struct BnRaw {
  static constexpr int P = V * sizeof(T) > 16 ? 16 / (int)sizeof(T) : V, BYTES = P * (int)sizeof(T);
  Vec<T, P> x[V / P];
  __device__ __forceinline__ void load(const BnRow<T>& row, int d) {
#pragma unroll
    for (int i = 0; i < V / P; ++i) {
      const int at = bn_col<V, WIDE>(d, i * P) * (int)sizeof(T);
      if constexpr (WIDE && BYTES == 16)
        x[i] = __builtin_bit_cast(Vec<T, P>, __builtin_amdgcn_raw_buffer_load_b128(row.r, at, 0, 0));
      else if constexpr (WIDE)
        x[i] = __builtin_bit_cast(Vec<T, P>, __builtin_amdgcn_raw_buffer_load_b64(row.r, at, 0, 0));
      else
#pragma unroll
        for (int j = 0; j < P; ++j) {
          if constexpr (sizeof(T) == 4)
            x[i].v[j] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(row.r, at + j * 64 * 4, 0, 0));
          else
            x[i].v[j] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(row.r, at + j * 64 * 2, 0, 0));
        }
    }
  }
  __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = to_f(x[j / P].v[j % P]);
  }
};
template <int V, bool WIDE>
__device__ __forceinline__ void bn_weights(float (&f)[V], const float* p, int d, int D) {
  BnRaw<V, WIDE, float> x;
  x.load(BnRow<float>(p, 0, D), d);
  x.get(f);
}
template <int V, bool WIDE, class T>
__device__ __forceinline__ void bn_put(const float (&f)[V], const BnRow<T>& row, int d) {
  using R = BnRaw<V, WIDE, T>;
#pragma unroll
  for (int i = 0; i < V; i += R::P) {
    const int at = bn_col<V, WIDE>(d, i) * (int)sizeof(T);
    Vec<T, R::P> x;
#pragma unroll
    for (int j = 0; j < R::P; ++j) x.v[j] = from_f<T>(f[i + j]);
    if constexpr (WIDE && R::BYTES == 16)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), row.r, at, 0, 0);
    else if constexpr (WIDE)
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), row.r, at, 0, 0);
    else
#pragma unroll
      for (int j = 0; j < R::P; ++j) {
        if constexpr (sizeof(T) == 4)
          __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x.v[j]), row.r, at + j * 64 * 4, 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, x.v[j]), row.r, at + j * 64 * 2, 0, 0);
      }
  }
}

// 1/sqrt(x) of a wave's one value: the instruction (1 ulp) where neither side leaves the normal numbers.
__device__ __forceinline__ float bn_rsqrt(float x) {
  return x > 0x1p-100f && x < 0x1p100f ? __builtin_amdgcn_rsqf(x) : 1.0f / sqrtf(x);
}

// act(g) and its derivative.  1 - sigmoid(g) is taken as exp(-g)*sigmoid(g) where the difference would cancel (at
// g = 10 it left 10 of 24 bits).
__device__ __forceinline__ float bn_act(int act, float g, float& d) {
  if (act == LSH_GATE_NONE) {
    d = 0.0f;
    return 1.0f;
  }
  const float e = __expf(-g), sg = __builtin_amdgcn_rcpf(1.0f + e);
  const float ds = sg * (g > 0.0f ? e * sg : 1.0f - sg);
  d = act == LSH_GATE_SILU ? __builtin_fmaf(g, ds, sg) : ds;
  return act == LSH_GATE_SILU ? g * sg : sg;
}

// A row is held in registers by W waves, E groups of V = 8 columns a lane: columns (e*64*W + lane)*8.
template <class TX, class TY, int W, int E, bool WIDE>
__global__ __launch_bounds__(W == 1 ? 256 : W * 64) void k_block_norm(BnArgs a) {
  constexpr int V = 8;
  __shared__ float s_red[2][W];
  const int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t row =
      W == 1 ? (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
  if (row >= a.rows) return;
  const float per = 1.0f / a.D;
  float xn[E][V], y[E][V], g[E][V];
  float r[1] = {0.0f};
  {
    BnRaw<V, WIDE, TX> rx[E];
    BnRaw<V, WIDE, TY> ry[E], rg[E];
    const BnRow<TX> bx(a.x, row, a.D);
    const BnRow<TY> by(a.y, row, a.D), bg(a.gate, row, a.D, a.act != LSH_GATE_NONE);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = (e * 64 * W + lane) * V;
      ry[e].load(by, d), rx[e].load(bx, d), rg[e].load(bg, d);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) ry[e].get(y[e]), rx[e].get(xn[e]), rg[e].get(g[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int j = 0; j < V; ++j) r[0] = __builtin_fmaf(y[e][j], y[e][j], r[0]);
  row_sums<W>(r, s_red[0]);
  const float ry = bn_rsqrt(r[0] * per + a.eps);
  r[0] = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = (e * 64 * W + lane) * V;
    float w[V], s[V];
    bn_weights<V, WIDE>(w, a.w_post, d, a.D);
    if (a.scale) bn_weights<V, WIDE>(s, a.scale, d, a.D);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float unused;
      const float act = a.act == LSH_GATE_NONE ? 1.0f : bn_act(a.act, g[e][j], unused);
      xn[e][j] = __builtin_fmaf(a.scale ? s[j] : a.scale1, act * (y[e][j] * ry * w[j]), xn[e][j]);
      r[0] = __builtin_fmaf(xn[e][j], xn[e][j], r[0]);
    }
    bn_put<V, WIDE>(xn[e], BnRow<TX>(a.x_new, row, a.D), d);
  }
  row_sums<W>(r, s_red[1]);
  const float rx = bn_rsqrt(r[0] * per + a.eps);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = (e * 64 * W + lane) * V;
    float w[V];
    bn_weights<V, WIDE>(w, a.w_pre, d, a.D);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] *= xn[e][j] * rx;
    bn_put<V, WIDE>(w, BnRow<TY>(a.z, row, a.D), d);
  }
}

// The gradients.  A workgroup takes rows blockIdx.x, + gridDim.x, ...; its sums of the parameters'
// gradients stay in registers until the last row and go to its place of `part`.  <m*y> needs dx, but with
// h = a*act*n it is <h*dx>/ry, whose sums do not, so a row has two reductions.
// HOLD: a row is read once, ahead, while the one before is worked on; without it (rows of more than 4096
// channels, which do not fit the registers) each sweep over the row reads it, mostly from the caches (bf16
// 2048 x 8192: 89 us, held 106 with spilled registers; 2048 x 16384: 196, with all sums in registers 417).
//
// What bounds it next to the bytes are the instructions a row (376 vector ones a wave of 64 x 4 columns):
// hence buffer accesses whose bounds replace selects and branches, sums over lanes without LDS, and a
// product with 1/D instead of a division.
template <class TX, class TY, int V, int W, int E, bool WIDE>
__global__ __launch_bounds__(W * 64) void k_block_norm_bwd(BnArgs a) {
  constexpr bool HOLD = E == 1;
  constexpr int K = HOLD ? E : 1;
  __shared__ float s_red[2][W * 5];
  // of the widest rows only one of the three sums has registers; a lane's other two lie in LDS
  constexpr bool LDS = E > 2;
  __shared__ Vec<float, V> s_sum[LDS ? 2 : 1][LDS ? E * W * 64 : 1];
  float sum[LDS ? 1 : 3][E][V] = {};
  if constexpr (LDS)
#pragma unroll
    for (int e = 0; e < E; ++e)
      s_sum[0][e * W * 64 + threadIdx.x] = s_sum[1][e * W * 64 + threadIdx.x] = Vec<float, V>{};
  BnRaw<V, WIDE, TX> qx[K], qgx[K];
  BnRaw<V, WIDE, TY> qy[K], qg[K], qgz[K];
  float x[K][V], y[K][V], g[K][V], gz[K][V], gx[K][V];
  const float per = 1.0f / a.D;
  // groups e.. of a row as read
  auto fetch = [&](int64_t row, int e) {
    const bool there = row < a.rows;
    const BnRow<TX> bx(a.x, row, a.D, there), bgx(a.gx, row, a.D, there && a.gx);
    const BnRow<TY> by(a.y, row, a.D, there), bgz(a.gz, row, a.D, there && a.gz);
    const BnRow<TY> bg(a.gate, row, a.D, there && a.act != LSH_GATE_NONE);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int d = ((e + k) * 64 * W + threadIdx.x) * V;
      qy[k].load(by, d), qx[k].load(bx, d), qg[k].load(bg, d), qgz[k].load(bgz, d), qgx[k].load(bgx, d);
    }
  };
  auto convert = [&] {
#pragma unroll
    for (int k = 0; k < K; ++k)
      qy[k].get(y[k]), qx[k].get(x[k]), qg[k].get(g[k]), qgz[k].get(gz[k]), qgx[k].get(gx[k]);
  };
  float wp[V], wq[V], sc[V];
  auto weights = [&](int e) {
    const int d = (e * 64 * W + threadIdx.x) * V;
    bn_weights<V, WIDE>(wp, a.w_post, d, a.D);
    bn_weights<V, WIDE>(wq, a.w_pre, d, a.D);
    if (a.scale)
      bn_weights<V, WIDE>(sc, a.scale, d, a.D);
    else
#pragma unroll
      for (int j = 0; j < V; ++j) sc[j] = a.scale1;
  };
  if (E == 1) weights(0);  // they stay
  if (HOLD) fetch(blockIdx.x, 0);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float r[1] = {0.0f};
    if constexpr (HOLD) {
      convert();
      fetch(row + gridDim.x, 0);
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int j = 0; j < V; ++j) r[0] = __builtin_fmaf(y[e][j], y[e][j], r[0]);
    } else {
      BnRaw<V, WIDE, TY> all[E];
#pragma unroll
      for (int e = 0; e < E; ++e) all[e].load(BnRow<TY>(a.y, row, a.D), (e * 64 * W + threadIdx.x) * V);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        all[e].get(y[0]);
#pragma unroll
        for (int j = 0; j < V; ++j) r[0] = __builtin_fmaf(y[0][j], y[0][j], r[0]);
      }
    }
    row_sums<W>(r, s_red[0]);
    const float ry = bn_rsqrt(r[0] * per + a.eps);
    float t[5] = {};  // of x_new^2, u*x_new, h*gx, h*u, h*x_new
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int k = HOLD ? e : 0;
      if (!HOLD) fetch(row, e), convert();
      if (E > 1) weights(e);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float unused;
        const float n = bn_act(a.act, g[k][j], unused) * (y[k][j] * ry * wp[j]);
        const float xn = __builtin_fmaf(sc[j], n, x[k][j]), h = sc[j] * n, u = gz[k][j] * wq[j];
        t[0] = __builtin_fmaf(xn, xn, t[0]);
        t[1] = __builtin_fmaf(u, xn, t[1]);
        t[2] = __builtin_fmaf(h, gx[k][j], t[2]);
        t[3] = __builtin_fmaf(h, u, t[3]);
        t[4] = __builtin_fmaf(h, xn, t[4]);
      }
    }
    row_sums<W>(t, s_red[1]);
    const float rx = bn_rsqrt(t[0] * per + a.eps);
    const float cx = rx * rx * (t[1] * per);
    const float cy = ry * ((t[2] + rx * (t[3] - cx * t[4])) * per);  // ry^2*<m*y>
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int k = HOLD ? e : 0, d = (e * 64 * W + threadIdx.x) * V;
      if (!HOLD) fetch(row, e), convert();
      if (E > 1) weights(e);
      Vec<float, V> s0, s1;
      if constexpr (LDS) s0 = s_sum[0][e * W * 64 + threadIdx.x], s1 = s_sum[1][e * W * 64 + threadIdx.x];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float dact;
        const float act = bn_act(a.act, g[k][j], dact);
        const float n = y[k][j] * ry * wp[j], xn = __builtin_fmaf(sc[j], act * n, x[k][j]);
        const float dx = gx[k][j] + rx * (gz[k][j] * wq[j] - xn * cx);
        const float dh = sc[j] * dx, dn = dh * act;
        float& sp = LDS ? s0.v[j] : sum[0][e][j];
        float& sq = LDS ? s1.v[j] : sum[LDS ? 0 : 1][e][j];
        float& sa = sum[LDS ? 0 : 2][e][j];
        sp = __builtin_fmaf(dn * y[k][j], ry, sp);
        sq = __builtin_fmaf(gz[k][j] * xn, rx, sq);
        sa = __builtin_fmaf(dx * act, n, sa);
        gx[k][j] = dx;
        g[k][j] = dh * n * dact;
        y[k][j] = ry * (dn * wp[j] - y[k][j] * cy);
      }
      if constexpr (LDS) s_sum[0][e * W * 64 + threadIdx.x] = s0, s_sum[1][e * W * 64 + threadIdx.x] = s1;
      bn_put<V, WIDE>(gx[k], BnRow<TX>(a.dx, row, a.D), d);
      bn_put<V, WIDE>(g[k], BnRow<TY>(a.dgate, row, a.D, a.dgate), d);
      bn_put<V, WIDE>(y[k], BnRow<TY>(a.dy, row, a.D), d);
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const BnRow<float> part(a.part, (int64_t)blockIdx.x * 3 + i, a.D);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = (e * 64 * W + threadIdx.x) * V;
      if (LDS && i < 2)
        bn_put<V, WIDE>(s_sum[i][LDS ? e * W * 64 + threadIdx.x : 0].v, part, d);
      else
        bn_put<V, WIDE>(sum[LDS ? 0 : i][e], part, d);
    }
  }
}

// dw_post, dw_pre and da: the workgroups' sums, kBnRuns runs of workgroups at once and then in run order.
// 768 workgroups' sums of 2048 channels (19 MB): 4.4 us, with 16 columns and 16 runs a workgroup 7.2.
constexpr int kBnCols = 32, kBnRuns = 32;
__global__ __launch_bounds__(kBnCols* kBnRuns) void k_block_norm_sums(const float* __restrict__ part, int P, int D,
                                                                     float* dw_post, float* dw_pre, float* da) {
  __shared__ float s_run[kBnRuns][kBnCols];
  const int c = threadIdx.x % kBnCols, run = threadIdx.x / kBnCols;
  const int i = blockIdx.x * kBnCols + c;
  const int per = (P + kBnRuns - 1) / kBnRuns, p1 = min(P, (run + 1) * per);
  float s = 0.0f;
  if (i < 3 * D)
#pragma unroll 8
    for (int p = run * per; p < p1; ++p) s += part[(size_t)p * 3 * D + i];
  s_run[run][c] = s;
  __syncthreads();
  if (run != 0 || i >= 3 * D) return;
  float* out = i < D ? dw_post : i < 2 * D ? dw_pre : da;
  if (!out) return;
  s = 0.0f;
#pragma unroll
  for (int r = 0; r < kBnRuns; ++r) s += s_run[r][c];
  out[i % D] = s;
}

// Calls f with values of the types of the residual stream and of the block.
template <class F>
static void with_types(int tx, int ty, F&& f) {
  with_dtype(ty, [&](auto y) {
    if (tx == LSH_F32)
      f(float{}, y);
    else
      f(y, y);
  });
}

// Calls f with the columns of a piece, the waves and the pieces a lane that hold D channels of a row.
//
// Forward: pieces of 8, which keep the row in registers between its sums.
//
// Gradients: what a wave does once a row (reductions, roots) is a third of its instructions with pieces of
// 4 and a sixth with 8, which take 158 registers instead of 91.  Rows of 257 to 2048 channels in wide
// accesses leave room for 3 waves a SIMD with 8 (bf16 8192 x 2048: 48 us, with 4 60).  Narrower rows would
// leave lanes idle, and element by element 8 take 190 registers.  Wider ones are one workgroup a CU, where 8 gain in
// some types what they lose in others (whole calls: bf16 4096 x 4096 101 us, with 4 103; 8192 x 2560 bf16 146 and 151,
// with an fp32 stream 180 and 171).  One workgroup a CU is also what bounds them: nothing runs while it waits at a
// row's two barriers (bf16 4096 x 4096 64 us and 4 for the sums, 2048 x 8192 89 and 6), and above 8192 channels 1024
// threads leave 128 registers, of which 6 to 64 too few (2048 x 16384: 196 and 10).
template <bool BWD, bool WIDE, class F>
static void with_row(int D, F&& f) {
  using std::integral_constant;
  const integral_constant<int, 4> v4;
  const integral_constant<int, 8> v8;
  const integral_constant<int, 16> v16;
  const integral_constant<int, 1> v1;
  const integral_constant<int, 2> v2;
  if constexpr (!BWD) {
    if (D <= 512)
      f(v8, v1, v1);
    else if (D <= 1024)
      f(v8, v2, v1);
    else if (D <= 2048)
      f(v8, v4, v1);
    else if (D <= 4096)
      f(v8, v8, v1);
    else if (D <= 8192)
      f(v8, v16, v1);
    else
      f(v8, v16, v2);
  } else {
    if (D <= 256)
      f(v4, v1, v1);
    else if (D <= 2048) {
      if constexpr (WIDE) {
        if (D <= 512)
          f(v8, v1, v1);
        else if (D <= 1024)
          f(v8, v2, v1);
        else
          f(v8, v4, v1);
      } else {
        if (D <= 512)
          f(v4, v2, v1);
        else if (D <= 1024)
          f(v4, v4, v1);
        else
          f(v4, v8, v1);
      }
    } else if (D <= 4096)
      f(v4, v16, v1);
    else if (D <= 8192)
      f(v4, v16, v2);
    else
      f(v4, v16, v4);
  }
}

static int bn_check(const lsh_block_norm* a) {
  if (!a || !lm_dtype_ok(a->x_dtype) || !lm_dtype_ok(a->dtype)) return LSH_ERR_ARG;
  if (a->x_dtype != LSH_F32 && a->x_dtype != a->dtype) return LSH_ERR_ARG;
  if (a->act < LSH_GATE_NONE || a->act > LSH_GATE_SIGMOID || !(a->eps >= 0.0f)) return LSH_ERR_ARG;
  if (a->rows < 0 || a->rows > 0x7fffffff || a->D < 1 || a->D > LSH_BLOCK_NORM_MAX_D) return LSH_ERR_SHAPE;
  if (a->rows > 0 && (bad_ptr(a->x) || bad_ptr(a->y) || bad_ptr(a->w_post) || bad_ptr(a->w_pre) ||
                      (a->act != LSH_GATE_NONE && bad_ptr(a->gate))))
    return LSH_ERR_ARG;
  return LSH_OK;
}

static BnArgs bn_args(const lsh_block_norm* p) {
  BnArgs a = {};
  a.x = p->x, a.y = p->y, a.gate = p->gate;
  a.w_post = p->w_post, a.w_pre = p->w_pre, a.scale = p->scale;
  a.scale1 = p->scale1, a.eps = p->eps, a.act = p->act, a.rows = p->rows, a.D = p->D;
  return a;
}

// Whether every row of every tensor begins at a multiple of 16 bytes.
static bool bn_wide(const BnArgs& a) {
  if (a.D % 8) return false;
  for (const void* p : {a.x, a.y, a.gate, (const void*)a.w_post, (const void*)a.w_pre, (const void*)a.scale,
                        (const void*)a.x_new, (const void*)a.z, a.gx, a.gz, (const void*)a.dx,
                        (const void*)a.dy, (const void*)a.dgate, (const void*)a.part})
    if ((uintptr_t)p % 16) return false;
  return true;
}

// Workgroups of the gradients, each with 3*D sums of its own: as many as the card holds at once with 12
// (pieces of 8) or 16 waves a CU.
static int64_t bn_grid(int64_t rows, int D, bool wide) {
  int64_t most;
  if (wide && D > 256 && D <= 2048)
    most = 256 * 12 / (D <= 512 ? 1 : D <= 1024 ? 2 : 4);
  else
    most = 256 * 16 / (D <= 256 ? 1 : D <= 512 ? 2 : D <= 1024 ? 4 : D <= 2048 ? 8 : 16);
  return rows < most ? rows : most;
}

}  // namespace lsh

using namespace lsh;

extern "C" int lsh_block_norm_fwd(const lsh_block_norm* p, void* x_new, void* z, void* stream) {
  if (int rc = bn_check(p)) return rc;
  if (p->rows == 0) return LSH_OK;
  if (bad_ptr(x_new) || bad_ptr(z)) return LSH_ERR_ARG;
  BnArgs a = bn_args(p);
  a.x_new = x_new, a.z = z;
  const bool wide = bn_wide(a);
  bool fits = true;
  with_types(p->x_dtype, p->dtype, [&](auto tx, auto ty) {
    with_row<false, true>(p->D, [&](auto, auto w, auto e) {
      using TX = decltype(tx);
      using TY = decltype(ty);
      constexpr int W = decltype(w)::value, E = decltype(e)::value;
      const dim3 grid((unsigned)(W == 1 ? (p->rows + 3) / 4 : p->rows));
      const int threads = W == 1 ? 256 : W * 64;
      fits = lm_grid_ok(grid.x, threads);
      if (!fits) return;
      if (wide)
        k_block_norm<TX, TY, W, E, true><<<grid, threads, 0, (hipStream_t)stream>>>(a);
      else
        k_block_norm<TX, TY, W, E, false><<<grid, threads, 0, (hipStream_t)stream>>>(a);
    });
  });
  if (!fits) return LSH_ERR_SHAPE;
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" size_t lsh_block_norm_bwd_workspace(const lsh_block_norm* p) {
  if (bn_check(p)) return 0;
  const int64_t wide = bn_grid(p->rows, p->D, p->D % 8 == 0), narrow = bn_grid(p->rows, p->D, false);
  return (size_t)(wide > narrow ? wide : narrow) * 3 * p->D * sizeof(float);
}

extern "C" int lsh_block_norm_bwd(const lsh_block_norm* p, const void* gx, const void* gz, void* dx,
                                  void* dy, void* dgate, float* dw_post, float* dw_pre, float* dscale,
                                  void* ws, size_t ws_bytes, void* stream) {
  if (int rc = bn_check(p)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const size_t need = lsh_block_norm_bwd_workspace(p);
  int64_t grid = 0;
  if (p->rows > 0) {
    if (bad_ptr(dx) || bad_ptr(dy)) return LSH_ERR_ARG;
    if (bad_ptr(ws) || ws_bytes < need) return LSH_ERR_WORKSPACE;
    BnArgs a = bn_args(p);
    a.gx = gx, a.gz = gz, a.dx = dx, a.dy = dy, a.dgate = dgate, a.part = (float*)ws;
    const bool wide = bn_wide(a);
    grid = bn_grid(p->rows, p->D, wide);
    with_types(p->x_dtype, p->dtype, [&](auto tx, auto ty) {
      using TX = decltype(tx);
      using TY = decltype(ty);
      auto go = [&](auto whole) {
        constexpr bool WIDE = decltype(whole)::value;
        with_row<true, WIDE>(p->D, [&](auto v, auto w, auto e) {
          constexpr int V = decltype(v)::value, W = decltype(w)::value, E = decltype(e)::value;
          k_block_norm_bwd<TX, TY, V, W, E, WIDE><<<dim3((unsigned)grid), W * 64, 0, st>>>(a);
        });
      };
      if (wide)
        go(std::true_type{});
      else
        go(std::false_type{});
    });
    LSH_CHECK_LAUNCH();
  }
  k_block_norm_sums<<<dim3((3 * p->D + kBnCols - 1) / kBnCols), kBnCols * kBnRuns, 0, st>>>(
      (const float*)ws, (int)grid, p->D, dw_post, dw_pre, dscale);
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
