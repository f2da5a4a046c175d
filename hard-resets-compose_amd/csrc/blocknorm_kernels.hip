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
// Bound by the rows' bytes; x_new is computed again instead of being kept.
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

// Sums over the lanes that share a row: one wave, or all W of the workgroup (through s, in wave order).
// One barrier: s is written again only after a barrier behind the next call's, which has another s.
template <int W, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* s) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum_f(v[i]);
  if constexpr (W > 1) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[w * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = s[i];
#pragma unroll
      for (int j = 1; j < W; ++j) v[i] += s[j * N + i];
    }
  }
}

// act(g) and its derivative
__device__ __forceinline__ float bn_act(int act, float g, float& d) {
  if (act == LSH_GATE_NONE) {
    d = 0.0f;
    return 1.0f;
  }
  const float sg = sigmoid_neg(g);
  const float ds = sg * (1.0f - sg);
  d = act == LSH_GATE_SILU ? __builtin_fmaf(g, ds, sg) : ds;
  return act == LSH_GATE_SILU ? g * sg : sg;
}

// A row is held in registers by W waves, E groups of V = 8 columns a lane: columns (e*64*W + lane)*8.
template <class TX, class TY, int W, int E, bool WIDE>
__global__ __launch_bounds__(W == 1 ? 256 : W * 64) void k_block_norm(BnArgs a) {
  constexpr int V = 8;
  __shared__ float s_red[2][W];
  const int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= a.rows) return;
  const size_t o = (size_t)row * a.D;
  float xn[E][V], y[E][V], g[E][V];
  float r[1] = {0.0f};
  {
    Raw<V, WIDE, TX> rx[E];
    Raw<V, WIDE, TY> ry[E], rg[E];
    const TY* gate = a.act != LSH_GATE_NONE ? (const TY*)a.gate : (const TY*)a.y;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = (e * 64 * W + lane) * V;
      ry[e].load((const TY*)a.y + o, d, a.D);
      rx[e].load((const TX*)a.x + o, d, a.D);
      rg[e].load(gate + o, d, a.D);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = (e * 64 * W + lane) * V;
      ry[e].get(y[e], d, a.D), rx[e].get(xn[e], d, a.D), rg[e].get(g[e], d, a.D);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int j = 0; j < V; ++j) r[0] = __builtin_fmaf(y[e][j], y[e][j], r[0]);
  row_sums<W>(r, s_red[0]);
  const float ry = 1.0f / sqrtf(r[0] / a.D + a.eps);
  r[0] = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = (e * 64 * W + lane) * V;
    float w[V], s[V];
    ld_vals<V, WIDE>(w, a.w_post, d, a.D);
    if (a.scale) ld_vals<V, WIDE>(s, a.scale, d, a.D);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float unused;
      const float act = a.act == LSH_GATE_NONE ? 1.0f : bn_act(a.act, g[e][j], unused);
      xn[e][j] = __builtin_fmaf(a.scale ? s[j] : a.scale1, act * (y[e][j] * ry * w[j]), xn[e][j]);
      r[0] = __builtin_fmaf(xn[e][j], xn[e][j], r[0]);
    }
    st_vals<V, WIDE>(xn[e], (TX*)a.x_new + o, d, a.D);
  }
  row_sums<W>(r, s_red[1]);
  const float rx = 1.0f / sqrtf(r[0] / a.D + a.eps);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = (e * 64 * W + lane) * V;
    float w[V];
    ld_vals<V, WIDE>(w, a.w_pre, d, a.D);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] *= xn[e][j] * rx;
    st_vals<V, WIDE>(w, (TY*)a.z + o, d, a.D);
  }
}

// The gradients.  A workgroup takes rows blockIdx.x, + gridDim.x, ...; its sums of the parameters'
// gradients stay in registers until the last row and go to its place of `part`.
template <class TX, class TY, int W, int E, bool WIDE>
__global__ __launch_bounds__(W * 64) void k_block_norm_bwd(BnArgs a) {
  constexpr int V = 4;  // with 8 the eight values a column take 168 registers: 8192 x 2048 197 us, not NN
  __shared__ float s_red[3][W * 2];
  float sum[3][E][V] = {};
  Raw<V, WIDE, TX> qx[E], qgx[E];
  Raw<V, WIDE, TY> qy[E], qg[E], qgz[E];
  // what is not there is read from what is, and not used
  const TY* gate = a.act != LSH_GATE_NONE ? (const TY*)a.gate : (const TY*)a.y;
  const TY* gzp = a.gz ? (const TY*)a.gz : (const TY*)a.y;
  const TX* gxp = a.gx ? (const TX*)a.gx : (const TX*)a.x;
  auto fetch = [&](int64_t row) {
    const size_t o = (size_t)row * a.D;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = (e * 64 * W + threadIdx.x) * V;
      qy[e].load((const TY*)a.y + o, d, a.D);
      qx[e].load((const TX*)a.x + o, d, a.D);
      qg[e].load(gate + o, d, a.D);
      qgz[e].load(gzp + o, d, a.D);
      qgx[e].load(gxp + o, d, a.D);
    }
  };
  fetch(blockIdx.x);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const size_t o = (size_t)row * a.D;
    float x[E][V], y[E][V], g[E][V], gz[E][V], gx[E][V];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = (e * 64 * W + threadIdx.x) * V;
      qy[e].get(y[e], d, a.D), qx[e].get(x[e], d, a.D), qg[e].get(g[e], d, a.D, a.act != LSH_GATE_NONE);
      qgz[e].get(gz[e], d, a.D, a.gz != nullptr), qgx[e].get(gx[e], d, a.D, a.gx != nullptr);
    }
    fetch(min(row + gridDim.x, a.rows - 1));  // while this row is worked on
    float r[1] = {0.0f};
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int j = 0; j < V; ++j) r[0] = __builtin_fmaf(y[e][j], y[e][j], r[0]);
    row_sums<W>(r, s_red[0]);
    const float ry = 1.0f / sqrtf(r[0] / a.D + a.eps);
    // x becomes x_new
    float t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = (e * 64 * W + threadIdx.x) * V;
      float wp[V], wq[V], s[V];
      ld_vals<V, WIDE>(wp, a.w_post, d, a.D);
      ld_vals<V, WIDE>(wq, a.w_pre, d, a.D);
      if (a.scale) ld_vals<V, WIDE>(s, a.scale, d, a.D);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float unused;
        const float act = bn_act(a.act, g[e][j], unused);
        x[e][j] = __builtin_fmaf(a.scale ? s[j] : a.scale1, act * (y[e][j] * ry * wp[j]), x[e][j]);
        t[0] = __builtin_fmaf(x[e][j], x[e][j], t[0]);
        t[1] = __builtin_fmaf(gz[e][j] * wq[j], x[e][j], t[1]);
      }
    }
    row_sums<W>(t, s_red[1]);
    const float rx = 1.0f / sqrtf(t[0] / a.D + a.eps);
    const float cx = rx * rx * (t[1] / a.D);
    // gx becomes dx, gz becomes dn
    r[0] = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = (e * 64 * W + threadIdx.x) * V;
      float wp[V], wq[V], s[V];
      ld_vals<V, WIDE>(wp, a.w_post, d, a.D);
      ld_vals<V, WIDE>(wq, a.w_pre, d, a.D);
      if (a.scale) ld_vals<V, WIDE>(s, a.scale, d, a.D);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float dx = gx[e][j] + rx * (gz[e][j] * wq[j] - x[e][j] * cx);
        float dact;
        const float act = bn_act(a.act, g[e][j], dact);
        const float n = y[e][j] * ry * wp[j], dh = (a.scale ? s[j] : a.scale1) * dx;
        sum[1][e][j] = __builtin_fmaf(gz[e][j] * x[e][j], rx, sum[1][e][j]);
        sum[2][e][j] = __builtin_fmaf(dx * act, n, sum[2][e][j]);
        gx[e][j] = dx;
        gz[e][j] = dh * act;
        g[e][j] = dh * n * dact;
        sum[0][e][j] = __builtin_fmaf(gz[e][j] * y[e][j], ry, sum[0][e][j]);
        r[0] = __builtin_fmaf(gz[e][j] * wp[j], y[e][j], r[0]);
      }
      st_vals<V, WIDE>(gx[e], (TX*)a.dx + o, d, a.D);
      if (a.dgate) st_vals<V, WIDE>(g[e], (TY*)a.dgate + o, d, a.D);
    }
    row_sums<W>(r, s_red[2]);
    const float cy = ry * ry * (r[0] / a.D);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = (e * 64 * W + threadIdx.x) * V;
      float wp[V];
      ld_vals<V, WIDE>(wp, a.w_post, d, a.D);
#pragma unroll
      for (int j = 0; j < V; ++j) wp[j] = ry * (gz[e][j] * wp[j] - y[e][j] * cy);
      st_vals<V, WIDE>(wp, (TY*)a.dy + o, d, a.D);
    }
  }
  float* part = a.part + (size_t)blockIdx.x * 3 * a.D;
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) st_vals<V, WIDE>(sum[i][e], part + (size_t)i * a.D, (e * 64 * W + threadIdx.x) * V, a.D);
}

// dw_post, dw_pre and da: the workgroups' sums, 16 runs of workgroups at once and then in run order.
__global__ __launch_bounds__(256) void k_block_norm_sums(const float* __restrict__ part, int P, int D,
                                                         float* dw_post, float* dw_pre, float* da) {
  __shared__ float s_run[16][16];
  const int c = threadIdx.x & 15, run = threadIdx.x >> 4;
  const int i = blockIdx.x * 16 + c;
  const int per = (P + 15) / 16, p1 = min(P, (run + 1) * per);
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
  for (int r = 0; r < 16; ++r) s += s_run[r][c];
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

// Calls f with the waves and the groups of PER columns a lane that hold D channels of a row.
template <int PER, class F>
static void with_row(int D, F&& f) {
  using std::integral_constant;
  const int lanes = (D + PER - 1) / PER;
  if (lanes <= 64)
    f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (lanes <= 128)
    f(integral_constant<int, 2>{}, integral_constant<int, 1>{});
  else if (lanes <= 256)
    f(integral_constant<int, 4>{}, integral_constant<int, 1>{});
  else if (lanes <= 512)
    f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  else if (lanes <= 1024)
    f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (lanes <= 2048)
    f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  else if constexpr (PER == 4)
    f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
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

// Workgroups of the gradients, each with 3*D sums of its own: 16 waves a CU.
static int64_t bn_grid(int64_t rows, int D) {
  const int64_t most = D <= 256 ? 4096 : D <= 512 ? 2048 : D <= 1024 ? 1024 : D <= 2048 ? 512 : 256;
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
  with_types(p->x_dtype, p->dtype, [&](auto tx, auto ty) {
    with_row<8>(p->D, [&](auto w, auto e) {
      using TX = decltype(tx);
      using TY = decltype(ty);
      constexpr int W = decltype(w)::value, E = decltype(e)::value;
      const dim3 grid((unsigned)(W == 1 ? (p->rows + 3) / 4 : p->rows));
      const int threads = W == 1 ? 256 : W * 64;
      if (wide)
        k_block_norm<TX, TY, W, E, true><<<grid, threads, 0, (hipStream_t)stream>>>(a);
      else
        k_block_norm<TX, TY, W, E, false><<<grid, threads, 0, (hipStream_t)stream>>>(a);
    });
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" size_t lsh_block_norm_bwd_workspace(const lsh_block_norm* p) {
  return bn_check(p) ? 0 : (size_t)bn_grid(p->rows, p->D) * 3 * p->D * sizeof(float);
}

extern "C" int lsh_block_norm_bwd(const lsh_block_norm* p, const void* gx, const void* gz, void* dx,
                                  void* dy, void* dgate, float* dw_post, float* dw_pre, float* dscale,
                                  void* ws, size_t ws_bytes, void* stream) {
  if (int rc = bn_check(p)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const size_t need = lsh_block_norm_bwd_workspace(p);
  const int64_t grid = bn_grid(p->rows, p->D);
  if (p->rows > 0) {
    if (bad_ptr(dx) || bad_ptr(dy)) return LSH_ERR_ARG;
    if (bad_ptr(ws) || ws_bytes < need) return LSH_ERR_WORKSPACE;
    BnArgs a = bn_args(p);
    a.gx = gx, a.gz = gz, a.dx = dx, a.dy = dy, a.dgate = dgate, a.part = (float*)ws;
    const bool wide = bn_wide(a);
    with_types(p->x_dtype, p->dtype, [&](auto tx, auto ty) {
      with_row<4>(p->D, [&](auto w, auto e) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        constexpr int W = decltype(w)::value, E = decltype(e)::value;
        if (wide)
          k_block_norm_bwd<TX, TY, W, E, true><<<dim3((unsigned)grid), W * 64, 0, st>>>(a);
        else
          k_block_norm_bwd<TX, TY, W, E, false><<<dim3((unsigned)grid), W * 64, 0, st>>>(a);
      });
    });
    LSH_CHECK_LAUNCH();
  }
  k_block_norm_sums<<<dim3((3 * p->D + 15) / 16), 256, 0, st>>>((const float*)ws, (int)grid, p->D, dw_post,
                                                              dw_pre, dscale);
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
