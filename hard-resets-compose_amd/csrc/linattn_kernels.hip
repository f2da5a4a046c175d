// Linear attention with a decay for each head, on MI355X (gfx950): a leaky integrator whose state
// is a matrix, the sibling of the LIF membrane (u = beta*u + x without the reset).
//
//   S_t = beta*S_{t-1} + k_t v_t^T          o_t = scale * q_t^T S_t
//
// Its gradients are the same recurrence.  With G_t = dL/dS_t and E_t = beta*G_t the part of it that
// reaches S_{t-1}:
//   dq_t = scale * S_t do_t
//   G_t  = E_{t+1} + scale * q_t do_t^T,    dk_t = G_t v_t,    dv_t = G_t^T k_t
// so dq is the forward walk with (do, v, k) in the place of (q, k, v) and the state transposed, and
// dk and dv are walks from the last row to the first with (v, do, q) and (k, q, do), which decay
// after the sum instead of before it.  One walk kernel therefore serves the forward and the
// backward: LaWalk names the operands by their place in the walk.
#include <algorithm>
#include <utility>

#include "lsh_lm.h"

namespace lsh {

// A [T, B, heads, D] operand: element strides of its rows, batches and heads (the last axis is
// contiguous), and how many of the walk's heads share one of its heads.
struct LaIn {
  const void* p;
  int64_t st, sb, sh;
  int share;
};

// One walk: out_r = so * Q_r^T S_r over the rows in walking order.
struct LaWalk {
  LaIn q, k, v;
  void* out;            // [T, B, H, DV], contiguous
  const float* s_in;    // [B*H] states of sk*DK or sv*DV elements, or NULL (zeros)
  float* s_out;         // the state after the last row, or NULL
  const float* beta;    // [H]
  int64_t T, B, H;
  int DK, DV;
  int sk, sv;           // element strides of a state along DK and DV
  int rev;              // rows from the last to the first
  int late;             // decay after the sum (gradient walks): S = beta*(S + K V^T)
  float so, su;         // out's scale, and the sum's
};

template <class T>
__device__ __forceinline__ const T* la_row(const LaIn& x, int64_t b, int64_t h) {
  return (const T*)x.p + b * x.sb + (h / x.share) * x.sh;
}

// One wave per state column: lane l holds rows l, l + 64, ... of column dv.
template <class T, class TO>
__global__ __launch_bounds__(256) void k_la_recur(LaWalk a) {
  const int lane = threadIdx.x & 63;
  const int dv = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (dv >= a.DV) return;
  const int64_t bh = blockIdx.x, b = bh / a.H, h = bh % a.H;
  const T* q = la_row<T>(a.q, b, h);
  const T* k = la_row<T>(a.k, b, h);
  const T* v = la_row<T>(a.v, b, h);
  TO* out = (TO*)a.out + (b * a.H + h) * a.DV + dv;
  const float beta = a.beta[h];
  const size_t state = (size_t)bh * a.DK * a.DV + (size_t)dv * a.sv;
  float S[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int dk = lane + 64 * i;
    S[i] = a.s_in && dk < a.DK ? a.s_in[state + (size_t)dk * a.sk] : 0.0f;
  }
  for (int64_t r = 0; r < a.T; ++r) {
    const int64_t t = a.rev ? a.T - 1 - r : r;
    const float vt = a.su * to_f(v[t * a.v.st + dv]);
    float o = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int dk = lane + 64 * i;
      if (dk < a.DK) {
        const float s = __builtin_fmaf(to_f(k[t * a.k.st + dk]), vt, a.late ? S[i] : beta * S[i]);
        o = __builtin_fmaf(to_f(q[t * a.q.st + dk]), s, o);
        S[i] = a.late ? beta * s : s;
      }
    }
    o = wave_sum_f(o);
    if (lane == 0) out[t * a.B * a.H * a.DV] = from_f<TO>(a.so * o);
  }
  if (a.s_out) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int dk = lane + 64 * i;
      if (dk < a.DK) a.s_out[state + (size_t)dk * a.sk] = S[i];
    }
  }
}

// Gradients of a shared head: the sum over the heads that share it, in fp32 and head order, from
// the walk's fp32 [rows, H, D] to [rows, H/share, D].
template <class T>
__global__ __launch_bounds__(256) void k_la_share(const float* __restrict__ x, T* __restrict__ y,
                                                  int64_t n, int D, int share) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const float* p = x + (i / D) * share * D + i % D;
  float s = 0.0f;
  for (int j = 0; j < share; ++j) s += p[(int64_t)j * D];
  y[i] = from_f<T>(s);
}

static int la_walk(const LaWalk& a, int dtype, bool out_f32, hipStream_t st) {
  if (a.B * a.H == 0) return LSH_OK;
  const dim3 grid((unsigned)(a.B * a.H), (a.DV + 3) / 4);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (out_f32)
      k_la_recur<T, float><<<grid, 256, 0, st>>>(a);
    else
      k_la_recur<T, T><<<grid, 256, 0, st>>>(a);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

// One token: the state is read, updated and written in place.  16 lanes cover 64 columns with
// 16-byte accesses, the 16 row groups of a workgroup take the state's rows in turn, and o is
// joined over the row groups in a fixed order.  Bound by the state's bytes.
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void k_la_step(LaIn qi, LaIn ki, LaIn vi,
                                                 const float* __restrict__ betas,
                                                 float* __restrict__ state, T* __restrict__ out,
                                                 int64_t H, int DK, int DV, float scale) {
  __shared__ float s_o[16][64 + 4];
  const int col = (threadIdx.x & 15) * 4, rg = threadIdx.x >> 4;
  const int dv0 = blockIdx.y * 64 + col;
  const int64_t bh = blockIdx.x, b = bh / H, h = bh % H;
  const T* q = la_row<T>(qi, b, h);
  const T* k = la_row<T>(ki, b, h);
  const T* v = la_row<T>(vi, b, h);
  const float beta = betas[h];
  float vt[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < 4; ++j) vt[j] = dv0 + j < DV ? to_f(v[dv0 + j]) : 0.0f;
  float* S = state + (size_t)bh * DK * DV + dv0;
  for (int dk = rg; dk < DK; dk += 16) {
    float* row = S + (size_t)dk * DV;
    const float kt = to_f(k[dk]), qt = to_f(q[dk]);
    if (WIDE) {
      if (dv0 < DV) {
        float4 s = *(float4*)row;
        s.x = __builtin_fmaf(kt, vt[0], beta * s.x);
        s.y = __builtin_fmaf(kt, vt[1], beta * s.y);
        s.z = __builtin_fmaf(kt, vt[2], beta * s.z);
        s.w = __builtin_fmaf(kt, vt[3], beta * s.w);
        *(float4*)row = s;
        o[0] = __builtin_fmaf(qt, s.x, o[0]);
        o[1] = __builtin_fmaf(qt, s.y, o[1]);
        o[2] = __builtin_fmaf(qt, s.z, o[2]);
        o[3] = __builtin_fmaf(qt, s.w, o[3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (dv0 + j < DV) {
          const float s = __builtin_fmaf(kt, vt[j], beta * row[j]);
          row[j] = s;
          o[j] = __builtin_fmaf(qt, s, o[j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s_o[rg][col + j] = o[j];
  __syncthreads();
  const int c = threadIdx.x;
  if (c < 64 && blockIdx.y * 64 + c < DV) {
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) sum += s_o[r][c];
    out[bh * DV + blockIdx.y * 64 + c] = from_f<T>(scale * sum);
  }
}

static int la_check(const lsh_linattn* a) {
  if (!a || !lm_dtype_ok(a->dtype)) return LSH_ERR_ARG;
  if (a->T < 0 || a->B < 0 || a->H < 0 || a->Dk < 1 || a->Dv < 1 || a->Dk > LSH_LINATTN_MAX_D ||
      a->Dv > LSH_LINATTN_MAX_D)
    return LSH_ERR_SHAPE;
  if (a->B * a->H > 0x7fffffff / 64 || a->T > ((int64_t)1 << 40)) return LSH_ERR_SHAPE;
  if (a->H > 0) {
    for (int n : {a->q_heads, a->k_heads, a->v_heads})
      if (n < 1 || a->H % n) return LSH_ERR_SHAPE;
    if (a->B > 0 && a->T > 0 && (bad_ptr(a->q) || bad_ptr(a->k) || bad_ptr(a->v) || bad_ptr(a->beta)))
      return LSH_ERR_ARG;
  }
  return LSH_OK;
}

static LaIn la_in(const void* p, int64_t st, int64_t sb, int64_t sh, int64_t H, int heads) {
  return LaIn{p, st, sb, sh, (int)(H / heads)};
}

}  // namespace lsh

using namespace lsh;

extern "C" int lsh_linattn_fwd(const lsh_linattn* a, void* stream) {
  if (int rc = la_check(a)) return rc;
  if (a->B == 0 || a->H == 0) return LSH_OK;
  if (a->T > 0 && bad_ptr(a->o)) return LSH_ERR_ARG;
  LaWalk w = {};
  w.q = la_in(a->q, a->q_st, a->q_sb, a->q_sh, a->H, a->q_heads);
  w.k = la_in(a->k, a->k_st, a->k_sb, a->k_sh, a->H, a->k_heads);
  w.v = la_in(a->v, a->v_st, a->v_sb, a->v_sh, a->H, a->v_heads);
  w.out = a->o;
  w.s_in = a->s0;
  w.s_out = a->s_end;
  w.beta = a->beta;
  w.T = a->T, w.B = a->B, w.H = a->H, w.DK = a->Dk, w.DV = a->Dv;
  w.sk = a->Dv, w.sv = 1;
  w.so = a->scale, w.su = 1.0f;
  return la_walk(w, a->dtype, false, (hipStream_t)stream);
}

extern "C" size_t lsh_linattn_bwd_workspace(const lsh_linattn* a) {
  if (la_check(a) || a->H == 0) return 0;
  size_t n = 0;
  for (auto [heads, D] : {std::pair<int, int>{a->q_heads, a->Dk}, {a->k_heads, a->Dk}, {a->v_heads, a->Dv}})
    if (heads != a->H) n = std::max(n, (size_t)a->T * a->B * a->H * D * 4);
  return n;
}

extern "C" int lsh_linattn_bwd(const lsh_linattn* a, const void* d_o, int64_t do_st, int64_t do_sb,
                               int64_t do_sh, const float* ds_end, void* dq, void* dk, void* dv,
                               float* ds0, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = la_check(a)) return rc;
  if (a->B == 0 || a->H == 0) return LSH_OK;
  if (a->T > 0 && (bad_ptr(d_o) || bad_ptr(dq) || bad_ptr(dk) || bad_ptr(dv))) return LSH_ERR_ARG;
  const size_t need = lsh_linattn_bwd_workspace(a);
  if (need && (bad_ptr(ws) || ws_bytes < need)) return LSH_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const LaIn q = la_in(a->q, a->q_st, a->q_sb, a->q_sh, a->H, a->q_heads);
  const LaIn k = la_in(a->k, a->k_st, a->k_sb, a->k_sh, a->H, a->k_heads);
  const LaIn v = la_in(a->v, a->v_st, a->v_sb, a->v_sh, a->H, a->v_heads);
  const LaIn d = la_in(d_o, do_st, do_sb, do_sh, a->H, (int)a->H);
  LaWalk w = {};
  w.beta = a->beta;
  w.T = a->T, w.B = a->B, w.H = a->H;
  auto run = [&](void* out, int heads) -> int {
    const bool shared = heads != a->H;
    w.out = shared ? ws : out;
    if (int rc = la_walk(w, a->dtype, shared, st)) return rc;
    if (shared && a->T > 0) {
      const int64_t n = a->T * a->B * heads * w.DV;
      with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        k_la_share<T><<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>((const float*)ws, (T*)out, n,
                                                                        w.DV, (int)(a->H / heads));
      });
      LSH_CHECK_LAUNCH();
    }
    return LSH_OK;
  };
  // dq: the forward walk with the state transposed
  w.q = d, w.k = v, w.v = k;
  w.DK = a->Dv, w.DV = a->Dk, w.sk = 1, w.sv = a->Dv;
  w.s_in = a->s0, w.so = a->scale, w.su = 1.0f;
  if (int rc = run(dq, a->q_heads)) return rc;
  // dk, from the last row
  w.q = v, w.k = d, w.v = q;
  w.rev = 1, w.late = 1, w.s_in = ds_end, w.so = 1.0f, w.su = a->scale;
  if (int rc = run(dk, a->k_heads)) return rc;
  // dv, and the gradient that leaves the first row
  w.q = k, w.k = q, w.v = d;
  w.DK = a->Dk, w.DV = a->Dv, w.sk = a->Dv, w.sv = 1, w.s_out = ds0;
  return run(dv, a->v_heads);
}

extern "C" int lsh_linattn_step(const lsh_linattn* a, float* state, void* stream) {
  if (int rc = la_check(a)) return rc;
  if (a->T != 1) return LSH_ERR_SHAPE;
  if (a->B == 0 || a->H == 0) return LSH_OK;
  if (bad_ptr(a->o) || bad_ptr(state)) return LSH_ERR_ARG;
  const LaIn q = la_in(a->q, 0, a->q_sb, a->q_sh, a->H, a->q_heads);
  const LaIn k = la_in(a->k, 0, a->k_sb, a->k_sh, a->H, a->k_heads);
  const LaIn v = la_in(a->v, 0, a->v_sb, a->v_sh, a->H, a->v_heads);
  const dim3 grid((unsigned)(a->B * a->H), (a->Dv + 63) / 64);
  const bool wide = a->Dv % 4 == 0 && (uintptr_t)state % 16 == 0;
  with_dtype(a->dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel) {
      kernel<<<grid, 256, 0, (hipStream_t)stream>>>(q, k, v, a->beta, state, (T*)a->o, a->H, a->Dk, a->Dv,
                                                   a->scale);
    };
    if (wide)
      go(k_la_step<T, true>);
    else
      go(k_la_step<T, false>);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
