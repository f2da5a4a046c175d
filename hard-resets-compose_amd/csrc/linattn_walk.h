// The chunked walk of linear attention (linattn_kernels.hip has the formulas): one workgroup takes a
// (batch, head), a block of state columns and a segment of rows, and walks the segment in chunks of C
// rows with the state in registers.  With r, s the rows of a chunk, n of them, and S the state before:
//
//   out_r = so * ( beta^(r+1) Q_r^T S + sum_{s<=r} beta^(r-s) (Q_r.K_s) V_s )
//   S'    = beta^n S + su * sum_s beta^(n-1-s) K_s V_s^T
//
// (walks that decay after the sum: beta^r and beta^(n-s); their scores carry su as well).
#pragma once
#include "lsh_lm.h"

namespace lsh {

// A [T, B, heads, D] operand: element strides of its rows, batches and heads (the last axis is
// contiguous), how many of the walk's heads share one of its heads, and whether its rows can be read
// 16 bytes at a time.
struct LaIn {
  const void* p;
  int64_t st, sb, sh;
  int share;
  bool wide;
};

// One walk: out_r = so * Q_r^T S_r over the rows in walking order.
struct LaWalk {
  LaIn q, k, v;
  void* out;            // [T, B, H, DV], contiguous
  bool out_f32;         // of fp32, whatever the operands' type
  const float* s_in;    // [segments, B*H] states before each segment, or NULL (zeros)
  float* s_out;         // the state after the last row, or NULL; of sums: see k_la_walk
  const float* beta;    // [H]
  int64_t T, B, H;
  int DK, DV;
  int sk, sv;           // element strides of a state along DK and DV
  int64_t L;            // rows of a segment, a multiple of the chunk when there are several
  int segs;
  int rev;              // rows from the last to the first
  int late;             // decay after the sum (gradient walks): S = beta*(S + K V^T)
  float so, su;         // out's scale, and the sum's
};

using f32x4 = float __attribute__((ext_vector_type(4)));
using bf16x4 = __bf16 __attribute__((ext_vector_type(4)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using s16x4 = short __attribute__((ext_vector_type(4)));

// What the matrix instructions take.  A fragment holds KB values of the summed axis for one of 16
// rows: lane l has row l%16 and, with g = l/16, the values 4g..4g+3 of each 16 (the order in which an
// accumulator holds its rows, so that an accumulator turns into a fragment in registers).
//
// bf16: products of bf16, fp32 sums.  fp32: the fp32 matrix instruction, exact products.  fp16 operands
// are computed in fp32: a state or a score can pass fp16's range where its result does not.
template <class L>
struct La;

template <>
struct La<bf16_t> {
  static constexpr int KB = 32, C = 64, TILES = 2;
  // a decayed value is taken in three bf16 parts, which hold its 24 bits: the state is kept to fp32
  static constexpr int PARTS = 3;
  using Frag = bf16x8;
  using Quad = bf16x4;
  static constexpr int kPadRow = 8, kPadCol = 16;  // elements; see the LDS layout at k_la_walk
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ Frag row(const bf16_t* p, int g) {
    const bf16x4 a = *(const bf16x4*)(p + 4 * g), b = *(const bf16x4*)(p + 16 + 4 * g);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // column l%16 of 32 rows: the LDS read that transposes blocks of 4 rows by 16 lanes
  static __device__ __forceinline__ Frag col(const bf16_t* p, int pitch, int g, int m) {
    using Lds = __attribute__((address_space(3))) s16x4*;
    const bf16_t* at = p + (4 * g + (m >> 2)) * pitch + (m & 3) * 4;
    const bf16x4 a = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)at));
    const bf16x4 b =
        __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(at + 16 * pitch)));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ Frag of(const f32x4* acc) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (bf16_t)acc[e >> 2][e & 3];
    return f;
  }
  static __device__ __forceinline__ int at(int e) { return (e >> 2) * 16 + (e & 3); }  // + 4g
};

template <>
struct La<float> {
  static constexpr int KB = 16, C = 32, TILES = 1, PARTS = 1;
  using Frag = f32x4;
  using Quad = f32x4;
  static constexpr int kPadRow = 4, kPadCol = 4;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag row(const float* p, int g) { return *(const f32x4*)(p + 4 * g); }
  static __device__ __forceinline__ Frag col(const float* p, int pitch, int g, int m) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = p[(4 * g + e) * pitch + m];
    return f;
  }
  static __device__ __forceinline__ Frag of(const f32x4* acc) { return acc[0]; }
  static __device__ __forceinline__ int at(int e) { return e; }
};

template <class T>
__device__ __forceinline__ const T* la_row(const LaIn& x, int64_t b, int64_t h) {
  return (const T*)x.p + b * x.sb + (h / x.share) * x.sh;
}

// 2^(n * log2 beta); l2 is finite (la_log2), so beta = 0 gives 1 for n = 0 and 0 beyond
__device__ __forceinline__ float la_pow(float l2, int n) { return __builtin_amdgcn_exp2f(l2 * (float)n); }
__device__ __forceinline__ float la_log2(float beta) { return fmaxf(log2f(beta), -1e4f); }

// A chunk of one operand on its way to LDS: C rows of DP columns (zeros beyond n rows and D columns),
// 16 bytes a piece, held in registers while the chunk before is worked on.
template <class T, class L, int C, int DP>
struct LaStage {
  static constexpr int W = kWide<T>, PER_ROW = DP / W, N = C * PER_ROW / 256;
  static_assert(C * PER_ROW % 256 == 0, "whole pieces for 256 threads");
  Vec<T, W> x[N];
  __device__ __forceinline__ void load(const T* base, int64_t st, bool wide, int D, int64_t t0, int rev,
                                       int n) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = threadIdx.x + 256 * i, r = u / PER_ROW, c = u % PER_ROW * W;
      const T* p = base + (rev ? t0 - r : t0 + r) * st + c;
      if (wide) {
        if (r < n && c < D) {
          x[i] = *(const Vec<T, W>*)p;
        } else {
#pragma unroll
          for (int j = 0; j < W; ++j) x[i].v[j] = (T)0.0f;
        }
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) x[i].v[j] = r < n && c + j < D ? p[j] : (T)0.0f;
      }
    }
  }
  __device__ __forceinline__ void put(L* lds, int pitch) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = threadIdx.x + 256 * i, r = u / PER_ROW, c = u % PER_ROW * W;
      Vec<L, W> y;
#pragma unroll
      for (int j = 0; j < W; ++j) y.v[j] = (L)x[i].v[j];
      constexpr int Q = kWide<L>;
#pragma unroll
      for (int j = 0; j < W; j += Q) *(Vec<L, Q>*)&lds[r * pitch + c + j] = *(Vec<L, Q>*)&y.v[j];
    }
  }
};

__device__ __forceinline__ bool la_odd(float x) { return !(fabsf(x) < INFINITY); }

// The walk.  SUMS: only the segments' sums (the state after each segment from a zero state before
// it), written to s_out [segments, B*H] one place further on (segment s to s + 1), for every segment
// but the last.
//
// Four waves; a wave owns NT*16 state columns and all DKP rows of them (the accumulators S), the four
// together a block of NT*64 columns.  Scores are computed once, their 16x16 tiles dealt to the waves,
// and shared through LDS.  All products are taken transposed (columns of the state by rows of the
// chunk), so scores, states and decayed values go from accumulator to operand in registers.
//
// LDS rows are padded: by 4 dwords modulo 64 where rows are read (16 rows of 8 or 16 bytes meet
// different banks), by 8 where the transposing read takes 8 rows of 32 bytes at once.
template <class T, class L, int DKP, int NT, bool SUMS>
__global__ __launch_bounds__(256, DKP <= 128 ? 2 : 1) void k_la_walk(LaWalk a) {
  using X = La<L>;
  using Frag = typename X::Frag;
  constexpr int C = X::C, KB = X::KB, DVB = NT * 64, KT = DKP / 16, CT = C / 16, KS = DKP / KB, CS = C / KB;
  constexpr int PQ = DKP + X::kPadRow, PK = DKP + X::kPadCol, PV = DVB + X::kPadCol, PP = C + X::kPadRow;
  __shared__ alignas(16) L s_q[SUMS ? 1 : C * PQ], s_k[C * PK], s_v[C * PV], s_p[SUMS ? 1 : C * PP];

  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  const int64_t BH = a.B * a.H;
  const int64_t seg = blockIdx.x / BH, bh = blockIdx.x % BH, b = bh / a.H, h = bh % a.H;
  const int dv0 = blockIdx.y * DVB, wc = w * NT * 16;  // the block's first column, the wave's within it
  const int64_t r0 = seg * a.L, r1 = min(a.T, r0 + a.L);
  const float l2 = la_log2(a.beta[h]);

  const T* q = la_row<T>(a.q, b, h);
  const T* k = la_row<T>(a.k, b, h);
  const T* v = la_row<T>(a.v, b, h) + dv0;

  const size_t size = (size_t)a.DK * a.DV;
  f32x4 S[KT][NT];
#pragma unroll
  for (int i = 0; i < KT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int dk = i * 16 + 4 * g + e, dv = dv0 + wc + t * 16 + m;
        S[i][t][e] = 0.0f;
        if (!SUMS && a.s_in && dk < a.DK && dv < a.DV)
          S[i][t][e] = a.s_in[(size_t)(seg * BH + bh) * size + (size_t)dk * a.sk + (size_t)dv * a.sv];
      }
  if (!SUMS) {
    for (int i = threadIdx.x; i < C * PP; i += 256) s_p[i] = (L)0.0f;  // tiles above the diagonal stay so
  }

  LaStage<T, L, C, DKP> xq, xk;
  LaStage<T, L, C, DVB> xv;
  auto fetch = [&](int64_t r) {
    const int n = (int)min((int64_t)C, r1 - r);
    const int64_t t0 = a.rev ? a.T - 1 - r : r;
    if (!SUMS) xq.load(q, a.q.st, a.q.wide, a.DK, t0, a.rev, n);
    xk.load(k, a.k.st, a.k.wide, a.DK, t0, a.rev, n);
    xv.load(v, a.v.st, a.v.wide, a.DV - dv0, t0, a.rev, n);
  };
  if (r0 < r1) fetch(r0);
  for (int64_t r = r0; r < r1; r += C) {
    const int n = (int)min((int64_t)C, r1 - r);
    __syncthreads();  // everyone has read the chunk before
    if (!SUMS) xq.put(s_q, PQ);
    xk.put(s_k, PK);
    xv.put(s_v, PV);
    __syncthreads();
    if (r + C < r1) fetch(r + C);

    f32x4 o[NT][CT];
    if (!SUMS) {
      // scores of rows 16i.. against rows 16j.., j <= i, with their decays
      int tile = 0;
#pragma unroll
      for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j, ++tile) {
          if ((tile & 3) != w) continue;
          f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int s = 0; s < KS; ++s)
            p = X::mma(X::row(&s_k[(j * 16 + m) * PK + s * KB], g), X::row(&s_q[(i * 16 + m) * PQ + s * KB], g), p);
          typename X::Quad y;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int far = (i - j) * 16 + m - 4 * g - e;
            y[e] = (L)(far >= 0 ? p[e] * (a.so * a.su) * la_pow(l2, far) : 0.0f);
          }
          *(typename X::Quad*)&s_p[(i * 16 + m) * PP + j * 16 + 4 * g] = y;
        }
      // what the state before the chunk gives
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < CT; ++i) o[t][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        Frag st[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          f32x4 x[X::TILES];
#pragma unroll
          for (int e = 0; e < X::TILES; ++e) x[e] = S[s * X::TILES + e][t];
          st[t] = X::of(x);
        }
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const Frag x = X::row(&s_q[(i * 16 + m) * PQ + s * KB], g);
#pragma unroll
          for (int t = 0; t < NT; ++t) o[t][i] = X::mma(st[t], x, o[t][i]);
        }
      }
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        const float f = a.so * la_pow(l2, i * 16 + m + 1 - a.late);
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][i] *= f;
      }
      __syncthreads();  // the scores are there
    }

    const float whole = la_pow(l2, n);
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) S[i][t] *= whole;
    bool odd = false;
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      Frag x[NT], part[NT][X::PARTS];
      float decay[KB / 4];
#pragma unroll
      for (int e = 0; e < KB / 4; ++e) {
        const int left = n - 1 - (s * KB + X::at(e) + 4 * g);
        decay[e] = left >= 0 ? a.su * la_pow(l2, left + a.late) : 0.0f;
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        x[t] = X::col(&s_v[s * KB * PV + wc + t * 16], PV, g, m);
#pragma unroll
        for (int e = 0; e < KB / 4; ++e) {
          const float y = (float)x[t][e];
          const bool bad = la_odd(y);
          odd |= bad;
          float rest = y * decay[e];
#pragma unroll
          for (int c = 0; c < X::PARTS; ++c) {
            const L top = (L)rest;
            part[t][c][e] = top;
            rest = bad ? 0.0f : rest - (float)top;
          }
          // a value that is not finite must not meet the zero scores of the rows before it
          if (bad) x[t][e] = (L)0.0f;
        }
      }
      if (!SUMS) {
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          if (s * X::TILES > i) continue;
          const Frag p = X::row(&s_p[(i * 16 + m) * PP + s * KB], g);
#pragma unroll
          for (int t = 0; t < NT; ++t) o[t][i] = X::mma(x[t], p, o[t][i]);
        }
      }
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const Frag y = X::col(&s_k[s * KB * PK + i * 16], PK, g, m);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < X::PARTS; ++c) S[i][t] = X::mma(y, part[t][c], S[i][t]);
      }
    }

    if (!SUMS) {
      if (wave_ballot(odd)) {
        // the values left out above, row by row for the rows from theirs on
        for (int j = 0; j < n; ++j)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = (float)s_v[j * PV + wc + t * 16 + 4 * g + e];
              if (la_odd(y))
#pragma unroll
                for (int i = 0; i < CT; ++i)
                  if (i * 16 + m >= j) o[t][i][e] += y * (float)s_p[(i * 16 + m) * PP + j];
            }
      }
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        if (i * 16 + m >= n) continue;
        const int64_t row = a.rev ? a.T - 1 - (r + i * 16 + m) : r + i * 16 + m;
        const size_t at = (size_t)(row * BH + bh) * a.DV;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int dv = dv0 + wc + t * 16 + 4 * g;
          if (dv >= a.DV) continue;
          const bool four = a.DV % 4 == 0;
          if (a.out_f32) {
            float* p = (float*)a.out + at + dv;
            if (four) {
              *(f32x4*)p = o[t][i];
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (dv + e < a.DV) p[e] = o[t][i][e];
            }
          } else {
            T* p = (T*)a.out + at + dv;
            Vec<T, 4> y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y.v[e] = from_f<T>(o[t][i][e]);
            if (four) {
              *(Vec<T, 4>*)p = y;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (dv + e < a.DV) p[e] = y.v[e];
            }
          }
        }
      }
    }
  }

  if (SUMS || (a.s_out && seg == a.segs - 1)) {
    float* to = a.s_out + (size_t)(SUMS ? (seg + 1) * BH + bh : bh) * size;
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int dk = i * 16 + 4 * g + e, dv = dv0 + wc + t * 16 + m;
          if (dk < a.DK && dv < a.DV) to[(size_t)dk * a.sk + (size_t)dv * a.sv] = S[i][t][e];
        }
  }
}

// Rows of a chunk for a dtype code, and columns of a workgroup's block for widths DK, DV.
inline int la_chunk(int dtype) { return dtype == LSH_BF16 ? La<bf16_t>::C : La<float>::C; }
inline int la_block(int DK, int DV) { return DK <= 128 && DV > 64 ? 128 : 64; }

// Launches the walk (its sums: SUMS) for operands of T computed in L.
template <class T, class L>
inline int la_launch(const LaWalk& a, bool sums, hipStream_t st) {
  const int64_t n = a.B * a.H * (sums ? a.segs - 1 : a.segs);
  if (n == 0) return LSH_OK;
  const int block = la_block(a.DK, a.DV);
  const dim3 grid((unsigned)n, (a.DV + block - 1) / block);
  auto go = [&](auto dkp, auto nt) {
    constexpr int DKP = decltype(dkp)::value, NT = decltype(nt)::value;
    if (sums)
      k_la_walk<T, L, DKP, NT, true><<<grid, 256, 0, st>>>(a);
    else
      k_la_walk<T, L, DKP, NT, false><<<grid, 256, 0, st>>>(a);
  };
  auto with = [&](auto dkp) {
    if (block == 128)
      go(dkp, std::integral_constant<int, 2>{});
    else
      go(dkp, std::integral_constant<int, 1>{});
  };
  if (a.DK <= 64)
    with(std::integral_constant<int, 64>{});
  else if (a.DK <= 128)
    with(std::integral_constant<int, 128>{});
  else
    go(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

int la_launch_f32(const LaWalk& a, bool sums, hipStream_t st);
int la_launch_bf16(const LaWalk& a, bool sums, hipStream_t st);
int la_launch_f16(const LaWalk& a, bool sums, hipStream_t st);

}  // namespace lsh
