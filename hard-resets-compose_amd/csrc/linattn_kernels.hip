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
// after the sum instead of before it.  One walk (linattn_walk.h) therefore serves the forward and the
// backward: LaWalk names the operands by their place in the walk.
#include <algorithm>
#include <utility>

#include "linattn_walk.h"

namespace lsh {

// The states before the segments from the segments' sums: starts[0] = s0 (or zeros), starts[s] =
// beta^L starts[s-1] + sum of segment s-1, in place.  One thread V elements, AHEAD segments' loads at once.
// Bound by the bytes where there are many heads (64 states of 128 x 128, 8 segments: 12.3 us for 62 MB, with one
// element a thread 16.0), by the chain of segments where there are few (8 of 64 x 128, 64 segments: one element
// and 16 ahead 9.0 us, with 8 ahead or four elements 1 to 2 more).
template <int V, int AHEAD>
__global__ __launch_bounds__(256) void k_la_join(float* __restrict__ starts, const float* __restrict__ s0,
                                                 const float* __restrict__ beta, int64_t n, int64_t size,
                                                 int64_t H, int segs, int64_t L) {
  using X = float __attribute__((ext_vector_type(V)));
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (i >= n) return;
  const float l2 = la_log2(beta[i / size % H]), f = __builtin_amdgcn_exp2f(l2 * (float)L);
  X s = s0 ? *(const X*)(s0 + i) : X(0.0f);
  *(X*)(starts + i) = s;
  for (int j0 = 1; j0 < segs; j0 += AHEAD) {
    X x[AHEAD];  // the loads first: one latency for several segments
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) x[j] = *(const X*)(starts + (size_t)min(j0 + j, segs - 1) * n + i);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        s[e] = f == INFINITY ? la_grow(s[e], l2, (float)L) + x[j][e] : __builtin_fmaf(f, s[e], x[j][e]);
      if (j0 + j < segs) *(X*)(starts + (size_t)(j0 + j) * n + i) = s;
    }
  }
}

// Gradients of shared heads: the sums over the heads that share one, in fp32 and head order, from the
// walks' fp32 [rows, H, D] to [rows, H/share, D].  Workgroups (., i) take operand i.
struct LaShares {
  const float* x[3];
  void* y[3];
  int64_t n[3];
  int D[3], share[3];
};
template <class T>
__global__ __launch_bounds__(256) void k_la_share(LaShares a) {
  const int j = blockIdx.y, D = a.D[j], share = a.share[j];
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.n[j]; i += (int64_t)gridDim.x * 256) {
    const float* p = a.x[j] + (i / D) * share * D + i % D;
    float s = 0.0f;
    for (int k = 0; k < share; ++k) s += p[(int64_t)k * D];
    ((T*)a.y[j])[i] = from_f<T>(s);
  }
}
constexpr int64_t kLaShareGroups = 1 << 20;  // at most; a grid has fewer than 2^32 threads

static int la_go(const LaWalks& all, int dtype, bool sums, hipStream_t st) {
  return dtype == LSH_F32    ? la_launch_f32(all, sums, st)
         : dtype == LSH_BF16 ? la_launch_bf16(all, sums, st)
                             : la_launch_f16(all, sums, st);
}
// Whether the walks' threads fit one launch.
static bool la_fits(const LaWalks& all, int dtype) {
  const LaWalk& a = all.w[0];
  const int block = la_block(dtype, a.DK, a.DV);
  return lm_grid_ok(a.B * a.H * a.segs * la_blocks(all, block) * all.n, block * 4);
}
static int la_go(const LaWalk& a, int dtype, bool sums, hipStream_t st) {
  LaWalks all = {};
  all.w[0] = a;
  all.n = 1;
  return la_go(all, dtype, sums, st);
}

// How the rows are split: every segment but the last has L rows.  The walk alone has a workgroup for
// each (batch, head) and block of columns; where these are too few for the chip the rows are split,
// at the price of a pass over K and V for the segments' sums and of their states.
struct LaSplit {
  int segs;
  int64_t L;
};
static LaSplit la_split(int dtype, int64_t T, int64_t BH, int DK, int DV) {
  const int64_t C = la_chunk(), chunks = (T + C - 1) / C;
  const int block = la_block(dtype, DK, DV);
  const int64_t groups = BH * ((DV + block - 1) / block);
  // LDS holds two workgroups a CU up to 128 state rows in 16 bits, up to 64 in fp32, and one above.  Measured with 256
  // and 512 workgroups, forward: bf16 4096 x 4 x 16 x 128 142 and 138 us, fp32 2048 x 4 x 16 x 128 152 and 169, bf16
  // 4096 x 16 x 256 x 256 130 and 147.
  const int64_t fill = std::max(DK, DV) <= (dtype == LSH_F32 ? 64 : 128) ? 512 : 256;
  int64_t segs = std::min<int64_t>((fill + groups - 1) / std::max<int64_t>(groups, 1), chunks / 2);
  if (segs < 2) return {1, std::max<int64_t>(T, 1)};
  const int64_t per = (chunks + segs - 1) / segs;
  return {(int)((chunks + per - 1) / per), per * C};
}

static void la_set_split(LaWalk& a, LaSplit s) { a.segs = s.segs, a.L = s.L; }

// The states before the segments (s.segs > 1), into `starts`.
static int la_starts(LaWalk a, int dtype, LaSplit s, const float* s0, float* starts, hipStream_t st) {
  la_set_split(a, s);
  a.s_in = nullptr;
  a.s_out = starts;
  if (int rc = la_go(a, dtype, true, st)) return rc;
  const int64_t size = (int64_t)a.DK * a.DV, n = a.B * a.H * size;
  auto join = [&](auto v, auto ahead) {
    constexpr int V = decltype(v)::value;
    k_la_join<V, decltype(ahead)::value><<<dim3((unsigned)((n + V * 256 - 1) / (V * 256))), 256, 0, st>>>(
        starts, s0, a.beta, n, size, a.H, s.segs, s.L);
  };
  if (n >= 1 << 19 && size % 4 == 0 && (uintptr_t)starts % 16 == 0 && (uintptr_t)s0 % 16 == 0)
    join(std::integral_constant<int, 4>{}, std::integral_constant<int, 8>{});
  else
    join(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

// One token: the state is read, updated and written in place.  16 lanes cover 64 columns, four a lane
// (WIDE: one 16-byte access, otherwise 16 columns apart), the 16 row groups of a workgroup take the
// state's rows in turn, and o is joined over the row groups in a fixed order.
// Bound by the state's bytes: 64 x 16 states of 128 x 128 22.5 us for 134 MB (6.0 TB/s, from the Infinity
// Cache); a single sequence by its launch (8 states of 64 x 64: 4 us).
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void k_la_step(LaIn qi, LaIn ki, LaIn vi,
                                                 const float* __restrict__ betas,
                                                 float* __restrict__ state, T* __restrict__ out,
                                                 int64_t H, int DK, int DV, float scale) {
  __shared__ float s_o[16][64 + 4];
  const int rg = threadIdx.x >> 4, col = (threadIdx.x & 15) * (WIDE ? 4 : 1);
  constexpr int STEP = WIDE ? 1 : 16;
  const int dv0 = blockIdx.y * 64 + col;
  const int64_t bh = blockIdx.x, b = bh / H, h = bh % H;
  const T* q = la_row<T>(qi, b, h);
  const T* k = la_row<T>(ki, b, h);
  const T* v = la_row<T>(vi, b, h);
  const float beta = betas[h] >= 0.0f ? betas[h] : NAN;  // as in the walks (la_log2)
  float vt[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < 4; ++j) vt[j] = dv0 + j * STEP < DV ? to_f(v[dv0 + j * STEP]) : 0.0f;
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
        if (dv0 + j * STEP < DV) {
          const float s = __builtin_fmaf(kt, vt[j], beta * row[j * STEP]);
          row[j * STEP] = s;
          o[j] = __builtin_fmaf(qt, s, o[j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s_o[rg][col + j * STEP] = o[j];
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
  if (!lm_grid_ok(a->B * a->H, 256) || a->T > ((int64_t)1 << 40)) return LSH_ERR_SHAPE;
  if (a->H > 0) {
    for (int n : {a->q_heads, a->k_heads, a->v_heads})
      if (n < 1 || a->H % n) return LSH_ERR_SHAPE;
    if (a->B > 0 && (bad_ptr(a->beta) || (a->T > 0 && (bad_ptr(a->q) || bad_ptr(a->k) || bad_ptr(a->v)))))
      return LSH_ERR_ARG;  // the decays are read without rows too
  }
  return LSH_OK;
}

static LaIn la_in(const void* p, int64_t st, int64_t sb, int64_t sh, int64_t H, int heads, int dtype, int D) {
  const int w = 16 / lm_dtype_size(dtype);
  const bool wide = (uintptr_t)p % 16 == 0 && st % w == 0 && sb % w == 0 && sh % w == 0 && D % w == 0;
  return LaIn{p, st, sb, sh, (int)(H / heads), wide};
}
static LaIn la_q(const lsh_linattn* a) {
  return la_in(a->q, a->q_st, a->q_sb, a->q_sh, a->H, a->q_heads, a->dtype, a->Dk);
}
static LaIn la_k(const lsh_linattn* a) {
  return la_in(a->k, a->k_st, a->k_sb, a->k_sh, a->H, a->k_heads, a->dtype, a->Dk);
}
static LaIn la_v(const lsh_linattn* a) {
  return la_in(a->v, a->v_st, a->v_sb, a->v_sh, a->H, a->v_heads, a->dtype, a->Dv);
}

// The split of the forward, and of its gradients' walks over the same rows.
static LaSplit la_split_of(const lsh_linattn* a) {
  return la_split(a->dtype, a->T, a->B * a->H, a->Dk, a->Dv);
}
static size_t la_starts_bytes(const lsh_linattn* a) {
  const LaSplit s = la_split_of(a);
  return s.segs > 1 ? (size_t)s.segs * a->B * a->H * a->Dk * a->Dv * sizeof(float) : 0;
}

}  // namespace lsh

using namespace lsh;

extern "C" size_t lsh_linattn_workspace(const lsh_linattn* a) {
  return la_check(a) || a->H == 0 ? 0 : la_starts_bytes(a);
}

extern "C" int lsh_linattn_fwd(const lsh_linattn* a, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = la_check(a)) return rc;
  if (a->B == 0 || a->H == 0) return LSH_OK;
  if (a->T > 0 && bad_ptr(a->o)) return LSH_ERR_ARG;
  const LaSplit split = la_split_of(a);
  if (split.segs > 1 && (bad_ptr(ws) || ws_bytes < la_starts_bytes(a))) return LSH_ERR_WORKSPACE;
  LaWalk w = {};
  w.q = la_q(a), w.k = la_k(a), w.v = la_v(a);
  w.out = a->o, w.out_f32 = a->dtype == LSH_F32;
  w.beta = a->beta;
  w.T = a->T, w.B = a->B, w.H = a->H, w.DK = a->Dk, w.DV = a->Dv;
  w.sk = a->Dv, w.sv = 1;
  w.so = a->scale, w.su = 1.0f;
  hipStream_t st = (hipStream_t)stream;
  if (split.segs > 1)
    if (int rc = la_starts(w, a->dtype, split, a->s0, (float*)ws, st)) return rc;
  la_set_split(w, split);
  w.s_in = split.segs > 1 ? (const float*)ws : a->s0;
  w.s_out = a->s_end;
  return la_go(w, a->dtype, false, st);
}

extern "C" size_t lsh_linattn_bwd_workspace(const lsh_linattn* a) {
  if (la_check(a) || a->H == 0) return 0;
  size_t n = 0;
  for (auto [heads, D] : {std::pair<int, int>{a->q_heads, a->Dk}, {a->k_heads, a->Dk}, {a->v_heads, a->Dv}})
    if (heads != a->H) n += (size_t)a->T * a->B * a->H * D * 4;
  return align_up(la_starts_bytes(a), 256) + n;
}

extern "C" int lsh_linattn_bwd(const lsh_linattn* a, const void* starts, const void* d_o, int64_t do_st,
                               int64_t do_sb, int64_t do_sh, const float* ds_end, void* dq, void* dk,
                               void* dv, float* ds0, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = la_check(a)) return rc;
  if (a->B == 0 || a->H == 0) return LSH_OK;
  if (a->T > 0 && (bad_ptr(d_o) || bad_ptr(dq) || bad_ptr(dk) || bad_ptr(dv))) return LSH_ERR_ARG;
  const LaSplit split = la_split_of(a);
  const size_t need = lsh_linattn_bwd_workspace(a);
  if ((need && (bad_ptr(ws) || ws_bytes < need)) || (split.segs > 1 && bad_ptr(starts)))
    return LSH_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  float* e_starts = (float*)ws;
  float* heads_f32 = (float*)((char*)ws + align_up(la_starts_bytes(a), 256));
  const LaIn q = la_q(a), k = la_k(a), v = la_v(a);
  const LaIn d = la_in(d_o, do_st, do_sb, do_sh, a->H, (int)a->H, a->dtype, a->Dv);
  LaWalk w = {};
  w.beta = a->beta;
  w.T = a->T, w.B = a->B, w.H = a->H;
  la_set_split(w, split);
  // a shared head's gradient is formed for every head that shares it, in fp32, and then summed
  struct Out {
    void* to;
    int heads;
    int D;
    float* f32;
  };
  auto out = [&](LaWalk& x, void* to, int heads) {
    const Out o = {to, heads, x.DV, heads != a->H ? heads_f32 : nullptr};
    x.out = o.f32 ? o.f32 : to;
    x.out_f32 = o.f32 || a->dtype == LSH_F32;
    if (o.f32) heads_f32 += (size_t)a->T * a->B * a->H * x.DV;
    return o;
  };
  // dv from the last row, and the gradient that leaves the first
  w.q = k, w.k = q, w.v = d;
  w.DK = a->Dk, w.DV = a->Dv, w.sk = a->Dv, w.sv = 1;
  w.rev = 1, w.late = 1, w.so = 1.0f, w.su = a->scale;
  if (split.segs > 1)
    if (int rc = la_starts(w, a->dtype, split, ds_end, e_starts, st)) return rc;
  w.s_in = split.segs > 1 ? e_starts : ds_end;
  LaWalk w_v = w, w_k = w, w_q = w;
  w_v.s_out = ds0;
  // dk, likewise with the state transposed
  w_k.q = v, w_k.k = d, w_k.v = q;
  w_k.DK = a->Dv, w_k.DV = a->Dk, w_k.sk = 1, w_k.sv = a->Dv;
  // dq: the forward walk with the state transposed
  w_q.q = d, w_q.k = v, w_q.v = k;
  w_q.DK = a->Dv, w_q.DV = a->Dk, w_q.sk = 1, w_q.sv = a->Dv;
  w_q.rev = w_q.late = 0, w_q.so = a->scale, w_q.su = 1.0f;
  w_q.s_in = split.segs > 1 ? (const float*)starts : a->s0;
  const Out outs[3] = {out(w_q, dq, a->q_heads), out(w_k, dk, a->k_heads), out(w_v, dv, a->v_heads)};
  LaWalks all = {};
  all.w[0] = w_q, all.w[1] = w_k, all.w[2] = w_v;
  const bool alike = la_rows(w_v.DK) == la_rows(w_q.DK) && la_block(a->dtype, w_v.DK, w_v.DV) == la_block(a->dtype, w_q.DK, w_q.DV);
  all.n = alike ? 3 : 2;
  if (la_fits(all, a->dtype)) {
    if (int rc = la_go(all, a->dtype, false, st)) return rc;
    if (!alike)
      if (int rc = la_go(w_v, a->dtype, false, st)) return rc;
  } else {  // more pairs than a launch of several walks has threads for: one after the other, as the forward's
    for (const LaWalk& x : all.w)
      if (int rc = la_go(x, a->dtype, false, st)) return rc;
  }
  LaShares shares = {};
  int count = 0;
  int64_t most = 0;
  for (const Out& o : outs) {
    if (!o.f32) continue;
    const int64_t n = a->T * a->B * o.heads * o.D;
    shares.x[count] = o.f32, shares.y[count] = o.to, shares.n[count] = n;
    shares.D[count] = o.D, shares.share[count++] = (int)(a->H / o.heads);
    most = most > n ? most : n;
  }
  if (most > 0) {
    const dim3 grid((unsigned)std::min((most + 255) / 256, kLaShareGroups), (unsigned)count);
    with_dtype(a->dtype, [&](auto t) { k_la_share<decltype(t)><<<grid, 256, 0, st>>>(shares); });
    LSH_CHECK_LAUNCH();
  }
  return LSH_OK;
}

extern "C" int lsh_linattn_step(const lsh_linattn* a, float* state, void* stream) {
  if (int rc = la_check(a)) return rc;
  if (a->T != 1) return LSH_ERR_SHAPE;
  if (a->B == 0 || a->H == 0) return LSH_OK;
  if (bad_ptr(a->o) || bad_ptr(state)) return LSH_ERR_ARG;
  const LaIn q = la_q(a), k = la_k(a), v = la_v(a);
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
