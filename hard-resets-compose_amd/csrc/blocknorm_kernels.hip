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
#include "lsh_lm.h"

namespace lsh {

constexpr int kBnThreads = 256;

template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float* s) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum_f(v[i]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) s[(threadIdx.x >> 6) * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.0f;
    for (int w = 0; w < kBnThreads / 64; ++w) v[i] += s[w * N + i];
  }
}

// act(g) and its derivative
__device__ __forceinline__ float bn_act(int act, float g, float& d) {
  if (act == LSH_GATE_NONE) {
    d = 0.0f;
    return 1.0f;
  }
  const float sg = 1.0f / (1.0f + expf(-g));
  const float ds = sg * (1.0f - sg);
  d = act == LSH_GATE_SILU ? __builtin_fmaf(g, ds, sg) : ds;
  return act == LSH_GATE_SILU ? g * sg : sg;
}

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

template <class TX, class TY>
__global__ __launch_bounds__(kBnThreads) void k_block_norm(BnArgs a) {
  __shared__ float s_red[kBnThreads / 64];
  const size_t o = (size_t)blockIdx.x * a.D;
  const TX* x = (const TX*)a.x + o;
  const TY* y = (const TY*)a.y + o;
  const TY* gate = (const TY*)a.gate + o;
  float r[1] = {0.0f};
  for (int d = threadIdx.x; d < a.D; d += kBnThreads) {
    const float v = to_f(y[d]);
    r[0] = __builtin_fmaf(v, v, r[0]);
  }
  block_sums(r, s_red);
  const float ry = 1.0f / sqrtf(r[0] / a.D + a.eps);
  auto next = [&](int d) {
    float unused;
    const float act = a.act == LSH_GATE_NONE ? 1.0f : bn_act(a.act, to_f(gate[d]), unused);
    const float n = to_f(y[d]) * ry * a.w_post[d];
    return __builtin_fmaf(a.scale ? a.scale[d] : a.scale1, act * n, to_f(x[d]));
  };
  r[0] = 0.0f;
  for (int d = threadIdx.x; d < a.D; d += kBnThreads) {
    const float v = next(d);
    r[0] = __builtin_fmaf(v, v, r[0]);
  }
  block_sums(r, s_red);
  const float rx = 1.0f / sqrtf(r[0] / a.D + a.eps);
  for (int d = threadIdx.x; d < a.D; d += kBnThreads) {
    const float v = next(d);
    ((TX*)a.x_new)[o + d] = from_f<TX>(v);
    ((TY*)a.z)[o + d] = from_f<TY>(v * rx * a.w_pre[d]);
  }
}

template <class TX, class TY>
__global__ __launch_bounds__(kBnThreads) void k_block_norm_bwd(BnArgs a) {
  __shared__ float s_red[kBnThreads / 64 * 2];
  float* part = a.part + (size_t)blockIdx.x * 3 * a.D;
  for (int d = threadIdx.x; d < 3 * a.D; d += kBnThreads) part[d] = 0.0f;
  __syncthreads();
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const size_t o = (size_t)row * a.D;
    const TX* x = (const TX*)a.x + o;
    const TY* y = (const TY*)a.y + o;
    const TY* gate = (const TY*)a.gate + o;
    const TX* gx = (const TX*)a.gx + o;
    const TY* gz = (const TY*)a.gz + o;
    float r[1] = {0.0f};
    for (int d = threadIdx.x; d < a.D; d += kBnThreads) {
      const float v = to_f(y[d]);
      r[0] = __builtin_fmaf(v, v, r[0]);
    }
    block_sums(r, s_red);
    const float ry = 1.0f / sqrtf(r[0] / a.D + a.eps);
    struct Row {
      float n, act, dact, s, xn, u;
    };
    auto at = [&](int d) {
      Row e;
      e.act = bn_act(a.act, a.act == LSH_GATE_NONE ? 0.0f : to_f(gate[d]), e.dact);
      e.n = to_f(y[d]) * ry * a.w_post[d];
      e.s = a.scale ? a.scale[d] : a.scale1;
      e.xn = __builtin_fmaf(e.s, e.act * e.n, to_f(x[d]));
      e.u = a.gz ? to_f(gz[d]) * a.w_pre[d] : 0.0f;
      return e;
    };
    float t[2] = {0.0f, 0.0f};
    for (int d = threadIdx.x; d < a.D; d += kBnThreads) {
      const Row e = at(d);
      t[0] = __builtin_fmaf(e.xn, e.xn, t[0]);
      t[1] = __builtin_fmaf(e.u, e.xn, t[1]);
    }
    block_sums(t, s_red);
    const float rx = 1.0f / sqrtf(t[0] / a.D + a.eps);
    const float cx = rx * rx * (t[1] / a.D);
    r[0] = 0.0f;
    auto grad_x = [&](const Row& e, int d) {
      return (a.gx ? to_f(gx[d]) : 0.0f) + rx * (e.u - e.xn * cx);
    };
    for (int d = threadIdx.x; d < a.D; d += kBnThreads) {
      const Row e = at(d);
      const float m = e.s * grad_x(e, d) * e.act * a.w_post[d];
      r[0] = __builtin_fmaf(m, to_f(y[d]), r[0]);
    }
    block_sums(r, s_red);
    const float cy = ry * ry * (r[0] / a.D);
    for (int d = threadIdx.x; d < a.D; d += kBnThreads) {
      const Row e = at(d);
      const float yd = to_f(y[d]), dx = grad_x(e, d), dh = e.s * dx, dn = dh * e.act;
      ((TX*)a.dx)[o + d] = from_f<TX>(dx);
      ((TY*)a.dy)[o + d] = from_f<TY>(ry * (dn * a.w_post[d] - yd * cy));
      if (a.dgate) ((TY*)a.dgate)[o + d] = from_f<TY>(dh * e.n * e.dact);
      part[d] += dn * yd * ry;
      if (a.gz) part[a.D + d] += to_f(gz[d]) * e.xn * rx;
      part[2 * a.D + d] += dx * e.act * e.n;
    }
  }
}

// dw_post, dw_pre and da: the workgroups' sums in workgroup order.
__global__ __launch_bounds__(256) void k_block_norm_sums(const float* __restrict__ part, int P, int D,
                                                         float* dw_post, float* dw_pre, float* da) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= 3 * D) return;
  float* out = i < D ? dw_post : i < 2 * D ? dw_pre : da;
  if (!out) return;
  float s = 0.0f;
  for (int p = 0; p < P; ++p) s += part[(size_t)p * 3 * D + i];
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

static int64_t bn_grid(int64_t rows) { return rows < 512 ? rows : 512; }

}  // namespace lsh

using namespace lsh;

extern "C" int lsh_block_norm_fwd(const lsh_block_norm* p, void* x_new, void* z, void* stream) {
  if (int rc = bn_check(p)) return rc;
  if (p->rows == 0) return LSH_OK;
  if (bad_ptr(x_new) || bad_ptr(z)) return LSH_ERR_ARG;
  BnArgs a = bn_args(p);
  a.x_new = x_new, a.z = z;
  with_types(p->x_dtype, p->dtype, [&](auto tx, auto ty) {
    k_block_norm<decltype(tx), decltype(ty)>
        <<<dim3((unsigned)p->rows), kBnThreads, 0, (hipStream_t)stream>>>(a);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" size_t lsh_block_norm_bwd_workspace(const lsh_block_norm* p) {
  return bn_check(p) ? 0 : (size_t)bn_grid(p->rows) * 3 * p->D * sizeof(float);
}

extern "C" int lsh_block_norm_bwd(const lsh_block_norm* p, const void* gx, const void* gz, void* dx,
                                  void* dy, void* dgate, float* dw_post, float* dw_pre, float* dscale,
                                  void* ws, size_t ws_bytes, void* stream) {
  if (int rc = bn_check(p)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const size_t need = lsh_block_norm_bwd_workspace(p);
  if (p->rows > 0) {
    if (bad_ptr(dx) || bad_ptr(dy)) return LSH_ERR_ARG;
    if (bad_ptr(ws) || ws_bytes < need) return LSH_ERR_WORKSPACE;
    BnArgs a = bn_args(p);
    a.gx = gx, a.gz = gz, a.dx = dx, a.dy = dy, a.dgate = dgate, a.part = (float*)ws;
    with_types(p->x_dtype, p->dtype, [&](auto tx, auto ty) {
      k_block_norm_bwd<decltype(tx), decltype(ty)>
          <<<dim3((unsigned)bn_grid(p->rows)), kBnThreads, 0, st>>>(a);
    });
    LSH_CHECK_LAUNCH();
  }
  k_block_norm_sums<<<dim3((3 * p->D + 255) / 256), 256, 0, st>>>((const float*)ws, (int)bn_grid(p->rows),
                                                                p->D, dw_post, dw_pre, dscale);
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
