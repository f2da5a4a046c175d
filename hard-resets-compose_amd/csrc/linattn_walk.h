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

// Walks of one size class that do not wait for each other.  Neighbouring workgroups take the n walks of a
// segment, which read some of the same operands and find them in the caches (bf16 4096 x 4 x 16 x 128: the
// three gradient walks with 23% fewer bytes from memory, 271 MB, than one walk after the other).
struct LaWalks {
  LaWalk w[3];
  int n;
};

using f32x4 = float __attribute__((ext_vector_type(4)));
using bf16x4 = __bf16 __attribute__((ext_vector_type(4)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x4 = _Float16 __attribute__((ext_vector_type(4)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using s16x4 = short __attribute__((ext_vector_type(4)));

// What the matrix instructions take.  A fragment holds KB values of the summed axis for one of 16
// rows: lane l has row l%16 and, with g = l/16, the values 4g..4g+3 of each 16 (the order in which an
// accumulator holds its rows, so that an accumulator turns into a fragment in registers).
//
// 16 bits: products of the type, fp32 sums.  What the walk holds in fp32 (a decayed value, a score, the state that
// meets q) is taken in parts: bf16 in three, which hold its 24 bits; fp16 in two, which hold 23 (one value in four
// is off by its last place).
// SCALED (fp16): what is split is first scaled by a power of two that brings its largest value below 2^15,
// since scores, states and decayed values can leave fp16's range, or sink below its normal numbers, where
// the results do not.
// fp32: the fp32 matrix instruction, exact products.
template <class L>
struct La;

template <class L, class F4, class F8>
struct La16 {
  static constexpr int KB = 32, C = 32, TILES = 2;
  using Frag = F8;
  using Quad = F4;
  static constexpr int kPadRow = 16, kPadCol = 16;  // elements; see the LDS layout at k_la_walk
  // a row's 32 values from their natural order, and from the order of packed()
  static __device__ __forceinline__ Frag row(const L* p, int g) {
    const F4 a = *(const F4*)(p + 4 * g), b = *(const F4*)(p + 16 + 4 * g);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ Frag packed_row(const L* p, int g) { return *(const Frag*)(p + 8 * g); }
  // where four values from c on lie when a fragment's eight are to be neighbours
  static __device__ __forceinline__ int packed(int c) { return (c & ~31) + (c & 12) * 2 + (c & 16) / 4; }
  // column l%16 of 32 rows: the LDS read that transposes blocks of 4 rows by 16 lanes
  static __device__ __forceinline__ Frag col(const L* p, int pitch, int g, int m) {
    using Lds = __attribute__((address_space(3))) s16x4*;
    const L* at = p + (4 * g + (m >> 2)) * pitch + (m & 3) * 4;
    const F4 a = __builtin_bit_cast(F4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)at));
    const F4 b = __builtin_bit_cast(F4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(at + 16 * pitch)));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ int at(int e) { return (e >> 2) * 16 + (e & 3); }  // + 4g
};

template <>
struct La<bf16_t> : La16<bf16_t, bf16x4, bf16x8> {
  static constexpr int PARTS = 3, FINE = 3;
  static constexpr bool SCALED = false;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // an accumulator's values as three fragments of eight bits each: the upper halves of the words, those of what
  // they leave, and the rest, which has no lower half
  static __device__ __forceinline__ void of(const f32x4* acc, float, Frag (&f)[3]) {
    unsigned top[3][4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float x = acc[e >> 2][e & 3], y = acc[e >> 2][(e & 3) + 1];
#pragma unroll
      for (int c = 0; c < 3; ++c) {
        const unsigned a = __builtin_bit_cast(unsigned, x), b = __builtin_bit_cast(unsigned, y);
        top[c][e / 2] = __builtin_amdgcn_perm(b, a, 0x07060302);
        x -= __builtin_bit_cast(float, a & 0xffff0000u);
        y -= __builtin_bit_cast(float, b & 0xffff0000u);
      }
    }
#pragma unroll
    for (int c = 0; c < 3; ++c) f[c] = __builtin_bit_cast(Frag, top[c]);
  }
};

template <>
struct La<f16_t> : La16<f16_t, f16x4, f16x8> {
  static constexpr int PARTS = 2, FINE = 2;
  static constexpr bool SCALED = true;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ void of(const f32x4* acc, float scale, Frag (&f)[2]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = acc[e >> 2][e & 3] * scale;
      f[0][e] = (f16_t)x;
      f[1][e] = (f16_t)(x - (float)f[0][e]);
    }
  }
  // the same over half a fragment: rows 16*half.. of the 32
  static __device__ __forceinline__ f32x4 mma_half(Frag a, Frag b, int half, f32x4 c) {
    const f16x4 x = half ? __builtin_shufflevector(a, a, 4, 5, 6, 7) : __builtin_shufflevector(a, a, 0, 1, 2, 3);
    const f16x4 y = half ? __builtin_shufflevector(b, b, 4, 5, 6, 7) : __builtin_shufflevector(b, b, 0, 1, 2, 3);
    return __builtin_amdgcn_mfma_f32_16x16x16f16(x, y, c, 0, 0, 0);
  }
};

// A power of two that scales a wave's values below 2^15, and its reciprocal.  Values that are not finite
// are left out: t holds a lane's largest of la_bits.
struct LaScale {
  float to, from;
};
__device__ __forceinline__ unsigned la_bits(float x) {  // grows with a finite |x|; 2^24 above its exponent
  return (__builtin_bit_cast(unsigned, x) << 1) + 0x01000000u;
}
__device__ __forceinline__ LaScale la_scale(unsigned t) {
  auto ror = [&](auto n) {
    const unsigned o = __builtin_amdgcn_update_dpp(t, t, 0x120 + decltype(n)::value, 0xf, 0xf, false);
    t = t > o ? t : o;
  };
  ror(std::integral_constant<int, 8>{});
  ror(std::integral_constant<int, 4>{});
  ror(std::integral_constant<int, 2>{});
  ror(std::integral_constant<int, 1>{});
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 64; i += 16) {
    const unsigned o = __builtin_amdgcn_readlane(t, i);
    top = top > o ? top : o;
  }
  const int e = min(max((int)(top >> 24) - 1, 15), 253);  // the exponent's bits
  return {__builtin_bit_cast(float, (unsigned)(268 - e) << 23), __builtin_bit_cast(float, (unsigned)(e - 14) << 23)};
}

template <>
struct La<float> {
  static constexpr int KB = 16, C = 32, TILES = 1, PARTS = 1, FINE = 1;
  static constexpr bool SCALED = false;
  using Frag = f32x4;
  using Quad = f32x4;
  static constexpr int kPadRow = 4, kPadCol = 4;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag row(const float* p, int g) { return *(const f32x4*)(p + 4 * g); }
  static __device__ __forceinline__ Frag packed_row(const float* p, int g) { return row(p, g); }
  static __device__ __forceinline__ int packed(int c) { return c; }
  static __device__ __forceinline__ Frag col(const float* p, int pitch, int g, int m) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = p[(4 * g + e) * pitch + m];
    return f;
  }
  static __device__ __forceinline__ void of(const f32x4* acc, float, Frag (&f)[1]) { f[0] = acc[0]; }
  static __device__ __forceinline__ int at(int e) { return e; }
};

template <class T>
__device__ __forceinline__ const T* la_row(const LaIn& x, int64_t b, int64_t h) {
  return (const T*)x.p + b * x.sb + (h / x.share) * x.sh;
}

// 2^(n * log2 beta); l2 is finite (la_log2), so beta = 0 gives 1 for n = 0 and 0 beyond.  What is no decay
// (below 0, or NaN) gives NaN.
__device__ __forceinline__ float la_pow(float l2, int n) { return __builtin_amdgcn_exp2f(l2 * (float)n); }
__device__ __forceinline__ float la_log2(float beta) { return beta >= 0.0f ? fmaxf(log2f(beta), -1e4f) : NAN; }
// x * 2^(l2 * n), l2 > 0, where the power alone may leave fp32: zeros stay zeros, and what fp32 holds is finite.
__device__ __forceinline__ float la_grow(float x, float l2, float n) {
  const float t = fminf(l2 * n, 1024.0f), whole = floorf(t);
  return __builtin_amdgcn_ldexpf(x * __builtin_amdgcn_exp2f(t - whole), (int)whole);
}

using u32x2 = unsigned __attribute__((ext_vector_type(2)));
using u32x4 = unsigned __attribute__((ext_vector_type(4)));

// Rows from a wave-uniform address on, by byte offsets below 2^31; kLaNowhere reads as zeros and is not
// written.
constexpr unsigned kLaNowhere = 0x80000000u;
struct LaRows {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ explicit LaRows(const void* base)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)kLaNowhere, 0x00020000)) {}
};

// A chunk of one operand on its way to LDS: C rows of DP columns, 16 bytes a piece, held in registers
// while the chunk before is worked on.  Row i of the n rows of a short chunk comes to row C - n + i, and
// the rows before it and the columns from D on are zeros: the distance to a chunk's end is the same in
// every chunk.  The loads have no branches around them (those cost the wait for all of them at the next
// loop head).  PACKED: in the order of La::packed.
template <class T, class L, int C, int DP, int THREADS, bool PACKED, bool WIDE>
struct LaStage {
  static constexpr int W = kWide<T>, PER_ROW = DP / W, ROWS = THREADS / PER_ROW;  // rows a piece of all threads
  static constexpr int N = C > ROWS ? C / ROWS : 1;
  static_assert(THREADS % PER_ROW == 0 && (C % ROWS == 0 || ROWS % C == 0), "whole rows");
  u32x4 x[N];
  const T* low;    // the lowest address of the chunk that is read next, as a whole one
  int64_t ahead;   // elements from a chunk to the next, `rows` rows on
  unsigned at;     // this thread's first piece, in bytes from low
  unsigned step;   // bytes from a row of the walk to the next, modulo 2^32 where it goes back
  int r0;
  __device__ __forceinline__ void init(const T* lowest, int64_t st, int rev, int D, int rows) {
    r0 = threadIdx.x / PER_ROW;
    low = lowest;
    ahead = rev ? -rows * st : rows * st;
    const unsigned bytes = (unsigned)st * (unsigned)sizeof(T);
    step = rev ? 0u - bytes : bytes;
    const int c = threadIdx.x % PER_ROW * W;
    at = (rev ? C - 1 - r0 : r0) * bytes + c * (unsigned)sizeof(T);
    if (c >= D || r0 >= C) at = kLaNowhere;
  }
  // the last n rows of the chunk at low
  __device__ __forceinline__ void load(int n) {
    const LaRows rows(low);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool there = at != kLaNowhere && r0 + i * ROWS >= C - n;
      x[i] = __builtin_amdgcn_raw_buffer_load_b128(rows.r, there ? at + i * ROWS * step : kLaNowhere, 0, 0);
    }
    low += ahead;
  }
  __device__ __forceinline__ void put(L* lds, int pitch) const {
    const int c = threadIdx.x % PER_ROW * W;
    if (ROWS > C && r0 >= C) return;
    constexpr int Q = PACKED ? 4 : kWide<L>;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Vec<T, W> z = __builtin_bit_cast(Vec<T, W>, x[i]);
      Vec<L, W> y;
#pragma unroll
      for (int j = 0; j < W; ++j) y.v[j] = (L)z.v[j];
#pragma unroll
      for (int j = 0; j < W; j += Q)
        *(Vec<L, Q>*)&lds[(r0 + i * ROWS) * pitch + (PACKED ? La<L>::packed(c + j) : c + j)] = *(Vec<L, Q>*)&y.v[j];
    }
  }
};

// n of eight 16-bit values fall out at the low end, zeros come in at the high end.
__device__ __forceinline__ u32x4 la_shift(u32x4 x, int n) {
  x = n & 8 ? u32x4{0, 0, 0, 0} : x;
  x = n & 4 ? u32x4{x[2], x[3], 0, 0} : x;
  x = n & 2 ? u32x4{x[1], x[2], x[3], 0} : x;
  return n & 1 ? u32x4{__builtin_amdgcn_alignbit(x[1], x[0], 16), __builtin_amdgcn_alignbit(x[2], x[1], 16),
                       __builtin_amdgcn_alignbit(x[3], x[2], 16), x[3] >> 16}
               : x;
}

// The same for operands whose rows do not begin at multiples of 16 bytes, or lie far apart.  Rows that are
// not there are read from one that is.
// 16 bits: a piece that would leave the row ends with it, and is shifted into place on its way to LDS (rows
// shorter than a piece are read element by element).  32 bits: element by element, a thread's columns
// PER_ROW apart, so that neighbouring lanes read neighbours.
// 4096 x 4 x 16 x 127 x 127 forward: bf16 175 us (128 columns 138), fp32 322 us (128 columns 275).  Element by element
// bf16 took half as long again, and fp32 in pieces a third.
template <class T, class L, int C, int DP, int THREADS, bool PACKED>
struct LaStage<T, L, C, DP, THREADS, PACKED, false> {
  static constexpr int W = kWide<T>, PER_ROW = DP / W, ROWS = THREADS / PER_ROW;
  static constexpr int N = C > ROWS ? C / ROWS : 1;
  static constexpr bool PIECES = sizeof(T) == 2;
  Vec<T, W> x[N];
  const T* low;
  int64_t ahead, step;  // elements, both signed
  int r0, D, first;     // rows from `first` on are there
  __device__ __forceinline__ void init(const T* lowest, int64_t st, int rev, int columns, int rows) {
    r0 = threadIdx.x / PER_ROW;
    step = rev ? -st : st;
    ahead = rows * step;
    low = rev ? lowest + (C - 1) * st : lowest;  // the chunk's row 0
    D = columns;
  }
  __device__ __forceinline__ void load(int n) {
    first = C - n;
    const T* from = n > 0 ? low : low - ahead;  // past the end, for good: the last chunk's last row again
    const int c = threadIdx.x % PER_ROW;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = r0 + i * ROWS;
      const T* row = from + (r >= first && r < C ? r : C - 1) * step;
      if (PIECES && D >= W)
        __builtin_memcpy(&x[i], row + min(c * W, D - W), 16);
      else
#pragma unroll
        for (int j = 0; j < W; ++j) x[i].v[j] = row[min(PIECES ? j : c + j * PER_ROW, D - 1)];
    }
    low = from + ahead;
  }
  __device__ __forceinline__ void put(L* lds, int pitch) const {
    if (ROWS > C && r0 >= C) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool there = r0 + i * ROWS >= first;
      L* row = lds + (r0 + i * ROWS) * pitch;
      if constexpr (PIECES) {
        const int c = threadIdx.x % PER_ROW * W;
        const int out = !there ? W : min(D >= W ? max(c - (D - W), 0) : c, W);
        const Vec<L, W> y = __builtin_bit_cast(Vec<L, W>, la_shift(__builtin_bit_cast(u32x4, x[i]), out));
        constexpr int Q = PACKED ? 4 : W;
#pragma unroll
        for (int j = 0; j < W; j += Q) {
          Vec<L, Q> z;
#pragma unroll
          for (int e = 0; e < Q; ++e) z.v[e] = c + j + e < D ? y.v[j + e] : (L)0.0f;
          *(Vec<L, Q>*)&row[PACKED ? La<L>::packed(c + j) : c + j] = z;
        }
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const int c = threadIdx.x % PER_ROW + j * PER_ROW;
          row[PACKED ? La<L>::packed(c & ~3) + (c & 3) : c] = there && c < D ? (L)x[i].v[j] : (L)0.0f;
        }
      }
    }
  }
};

__device__ __forceinline__ bool la_odd(float x) { return !(fabsf(x) < INFINITY); }

// Four columns of the chunk's rows i*16 + m to the output, o[i] to byte at + i*16*step (modulo 2^32) from low.
template <class TO, int CT>
__device__ __forceinline__ void la_store(TO* low, unsigned at, unsigned step, const f32x4 (&o)[CT],
                                         int first) {
  const LaRows rows(low);
#pragma unroll
  for (int i = 0; i < CT; ++i) {
    Vec<TO, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = from_f<TO>(o[i][e]);
    const unsigned b = at != kLaNowhere && i * 16 >= first ? at + i * 16 * step : kLaNowhere;
    if constexpr (sizeof(TO) == 4)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), rows.r, b, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, y), rows.r, b, 0, 0);
  }
}
// The same where rows begin anywhere: p is row m's first column, left of them are there.
template <class TO, int CT>
__device__ __forceinline__ void la_store_some(TO* p, int64_t step, const f32x4 (&o)[CT], int first, int left) {
#pragma unroll
  for (int i = 0; i < CT; ++i) {
    if (i * 16 < first) continue;
    Vec<TO, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = from_f<TO>(o[i][e]);
    if (left >= 4)
      __builtin_memcpy(p + i * 16 * step, &y, sizeof(y));
    else
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) p[i * 16 * step + e] = y.v[e];
  }
}

// Whether any of a fragment's values is not finite: the exponent's bits, plus one in their last place; all
// ones carry into the bit above.
__device__ __forceinline__ bool la_odd(u32x4 b, unsigned exponents, unsigned one) {
  unsigned any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= (b[i] & exponents) + one;
  return (any & 0x80008000u) != 0;
}
__device__ __forceinline__ bool la_odd(bf16x8 x) {
  return la_odd(__builtin_bit_cast(u32x4, x), 0x7f807f80u, 0x00800080u);
}
__device__ __forceinline__ bool la_odd(f16x8 x) {
  return la_odd(__builtin_bit_cast(u32x4, x), 0x7c007c00u, 0x04000400u);
}
__device__ __forceinline__ bool la_odd(f32x4 x) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= la_odd(x[i]);
  return any;
}

// Waves a SIMD that LDS has room for.
constexpr int la_waves(int size, int DKP, int W) {
  return DKP > 128 ? W / 4 : size == 4 ? DKP > 64 ? W / 4 : 2 : W == 8 ? 4 : 2;
}

// The walk.  SUMS: only the segments' sums (the state after each segment from a zero state before
// it), written to s_out [segments, B*H] one place further on (segment s to s + 1), for every segment
// but the last.  WIDE: every row is read and written in whole pieces (la_wide).
//
// W waves; a wave owns 16 state columns and all DKP rows of them (the accumulators S).  Scores are
// computed once, their 16x16 tiles dealt to the waves, and shared through LDS.  All products are taken
// transposed (columns of the state by rows of the chunk), so scores, states and decayed values go from
// accumulator to operand in registers.
//
// LDS rows are padded by 8 dwords modulo 64 (fp32: by 4), so that the 16 rows of 16 bytes of a fragment, and
// the 8 rows of 32 bytes that the transposing read takes at once, meet different banks.  Where rows are read
// 4 dwords gave twice the conflicts (3.2 -> 6.0 million cycles of the forward walk below) and 1% of time.
//
// Bound by the vector instructions, the bytes and the latency of a chunk's steps between its barriers: bf16,
// 4096 x 4 x 16 x 128, forward 88 us for 302 MB with the states (3.4 TB/s; 8 us pass until the first chunk and state
// arrive), the gradients' three walks 230 us for 905 MB (3.9 TB/s).  Of a SIMD's cycles 53% issue vector instructions
// (gradients 66%) and 28% keep the matrix unit busy (35%); nearly half of the vector instructions take the state apart
// for q.  With two parts for scores and that state the walks take 78 and 200 us, but hold 16 of fp32's 24 bits.
// fp16 103 and 270 us.  fp32 192 and 554 us, with the matrix unit busy for 67% and 71% of it.
template <class T, class L, int DKP, int W, bool SUMS, bool WIDE>
__global__ __launch_bounds__(W * 64, la_waves(sizeof(L), DKP, W)) void k_la_walk(LaWalks all) {
  const int64_t turn = xcd_neuron(blockIdx.x, gridDim.x), job = turn / all.n;
  const LaWalk& a = all.w[turn % all.n];
  using X = La<L>;
  using Frag = typename X::Frag;
  constexpr int C = X::C, KB = X::KB, DVB = W * 16, KT = DKP / 16, CT = C / 16, KS = DKP / KB, CS = C / KB;
  static_assert(CT * (CT + 1) / 2 <= W, "a wave has one tile of the scores at most");
  constexpr int PQ = DKP + X::kPadRow, PK = DKP + X::kPadCol, PV = DVB + X::kPadCol, PP = C + X::kPadRow;
  // of each two halves: one is filled while the other is read
  __shared__ alignas(16) L s_q[SUMS ? 8 : 2 * C * PQ], s_k[2 * C * PK], s_v[2 * C * PV];
  __shared__ alignas(16) L s_p[X::FINE][SUMS ? 8 : C * PP];
  __shared__ float s_from[W];  // SCALED: what takes each tile of the scores back

  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t BH = a.B * a.H;
  const int blocks = (a.DV + DVB - 1) / DVB;
  const int64_t pair = job / blocks;
  const int64_t seg = pair / BH, bh = pair % BH, b = bh / a.H, h = bh % a.H;
  if (seg >= a.segs - SUMS) return;  // another walk of the launch has more blocks
  const int dv0 = (int)(job % blocks) * DVB, wc = w * 16;  // the block's first column, the wave's within it
  const int64_t r0 = seg * a.L, r1 = min(a.T, r0 + a.L);
  const T* q = la_row<T>(a.q, b, h);
  const T* k = la_row<T>(a.k, b, h);
  const T* v = la_row<T>(a.v, b, h) + dv0;

  // state element (i*16 + 4g + e, m) of the wave's columns is at i*16*sk + e*sk from here
  const size_t size = (size_t)a.DK * a.DV;
  int at0 = 4 * g * a.sk + (dv0 + wc + m) * a.sv;
  const bool col = dv0 + wc + m < a.DV;
  f32x4 S[KT];
  {
    const float* from = a.s_in + (size_t)(seg * BH + bh) * size;
    if (!SUMS && a.s_in && a.sk == 1 && a.DK % 4 == 0) {
#pragma unroll
      for (int i = 0; i < KT; ++i)
        S[i] = col && i * 16 + 4 * g < a.DK ? *(const f32x4*)(from + at0 + i * 16) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    } else {
#pragma unroll
      for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          S[i][e] = 0.0f;
          if (!SUMS && a.s_in && col && i * 16 + 4 * g + e < a.DK) S[i][e] = from[at0 + (i * 16 + e) * a.sk];
        }
    }
  }
  // the state is sigma*S: most chunks decay it by sigma alone, and weigh what they add by 1/sigma.  sigma is a power
  // of its own, not a product of the chunks' (whose one rounding would come again in every chunk: 6.5e-6 after 512).
  float sigma = 1.0f;
  int since = 0;  // the rows that sigma stands for
  if (!SUMS) {
    for (int i = threadIdx.x; i < X::FINE * C * PP; i += W * 64) s_p[0][i] = (L)0.0f;  // tiles above the diagonal stay so
  }

  // A chunk's powers reach beta^C, and sigma adds to them: with beta = 4 less than 2^81.  Heads that grow faster take
  // one row at a time, as if each were a short chunk, so that no power is formed that overflows where the results
  // do not (beta^31 of rows that hold zeros, or are not there).
  const float l2 = la_log2(a.beta[h]);
  const int step = __builtin_amdgcn_readfirstlane(l2 > 2.0f ? 1 : C);
  // row r of the walk is row (rev ? T - 1 - r : r); the first chunk is the short one
  int n = r0 < r1 ? step == 1 ? 1 : (int)((r1 - r0 - 1) % C) + 1 : 0;
  int64_t r = r0 + n - C;  // where the chunk's row 0 would be
  float decay[CS][KB / 4];  // of the rows to the chunk's end; where step is 1, of the last row only
#pragma unroll
  for (int s = 0; s < CS; ++s)
#pragma unroll
    for (int e = 0; e < KB / 4; ++e) {
      const int left = C - 1 - (s * KB + X::at(e) + 4 * g);
      decay[s][e] = left < step ? a.su * la_pow(l2, left + a.late) : 0.0f;
    }
  // this wave's tile of the scores: rows 16*ti + m against rows 16*tj + 4g + e
  const int ti = w == 0 ? 0 : w < 3 ? 1 : w < 6 ? 2 : 3, tj = w - ti * (ti + 1) / 2;
  float fall[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int far = max((ti - tj) * 16 + m - 4 * g - e, 0);
    fall[e] = far < step ? a.so * a.su * la_pow(l2, far) : 0.0f;
  }

  LaStage<T, L, C, DKP, W * 64, true, WIDE> xq;
  LaStage<T, L, C, DKP, W * 64, false, WIDE> xk;
  LaStage<T, L, C, DVB, W * 64, false, WIDE> xv;
  auto fetch = [&](int n) {
    if (!SUMS) xq.load(n);
    xk.load(n);
    xv.load(n);
  };
  auto put = [&](int half) {
    if (!SUMS) xq.put(s_q + half * (C * PQ), PQ);
    xk.put(s_k + half * (C * PK), PK);
    xv.put(s_v + half * (C * PV), PV);
  };
  const int64_t so = BH * a.DV;  // elements from a row of the output to the next
  const int dv = dv0 + wc + 4 * g;
  // the lowest address of the chunk's output, this lane's first byte from there, and bytes to the next row
  const int64_t low = a.rev ? a.T - r - C : r;  // the chunk's row of lowest address
  const unsigned eo = a.out_f32 ? 4 : sizeof(T), bo = (unsigned)so * eo, step_o = a.rev ? 0u - bo : bo;
  const int64_t ahead_o = (a.rev ? -step : step) * so * eo;
  char* out = (char*)a.out + ((low * BH + bh) * a.DV + dv0) * eo;
  const unsigned at_o = dv < a.DV ? (a.rev ? C - 1 - m : m) * bo + (wc + 4 * g) * eo : kLaNowhere;
  xq.init(q + low * a.q.st, a.q.st, a.rev, a.DK, step);
  xk.init(k + low * a.k.st, a.k.st, a.rev, a.DK, step);
  xv.init(v + low * a.v.st, a.v.st, a.rev, a.DV - dv0, step);
  if (n) {
    fetch(n);
    put(0);
    fetch(r + C + step <= r1 ? step : 0);
  }
  __syncthreads();
  int half = 0;
  for (; n && r + C <= r1; r += step, n = step) {
    const L *cq = s_q + half * (C * PQ), *ck = s_k + half * (C * PK), *cv = s_v + half * (C * PV);
    Frag x[CS];  // the chunk's values in the wave's columns
#pragma unroll
    for (int s = 0; s < CS; ++s) x[s] = X::col(&cv[s * KB * PV + wc], PV, g, m);
    if (!SUMS) {
      // scores with their decays
      if (w < CT * (CT + 1) / 2) {
        f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s)
          p = X::mma(X::row(&ck[(tj * 16 + m) * PK + s * KB], g), X::packed_row(&cq[(ti * 16 + m) * PQ + s * KB], g), p);
        typename X::Quad y;
        unsigned big = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = (ti - tj) * 16 + m - 4 * g - e >= 0 ? p[e] * fall[e] : 0.0f;
          big = max(big, la_bits(p[e]));
        }
        if constexpr (X::SCALED) {
          const LaScale c = la_scale(big);
          p *= c.to;
          if (lane == 0) s_from[w] = c.from;
        }
#pragma unroll
        for (int c = 0; c < X::FINE; ++c) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = (L)p[e];
            p[e] -= (float)y[e];
          }
          *(typename X::Quad*)&s_p[c][(ti * 16 + m) * PP + X::packed(tj * 16 + 4 * g)] = y;
        }
      }
      // what the state before the chunk gives
      f32x4 o[CT];
#pragma unroll
      for (int i = 0; i < CT; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      LaScale in = {1.0f, 1.0f};
      if constexpr (X::SCALED) {
        unsigned big = 0;
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) big = max(big, la_bits(S[i][e]));
        in = la_scale(big);
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        Frag st[X::FINE];
        X::of(&S[s * X::TILES], in.to, st);
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const Frag y = X::packed_row(&cq[(i * 16 + m) * PQ + s * KB], g);
#pragma unroll
          for (int c = 0; c < X::FINE; ++c) o[i] = X::mma(st[c], y, o[i]);
        }
      }
      const int first = C - n - m;  // a lane's rows of the chunk are those with 16i >= first
#pragma unroll
      for (int i = 0; i < CT; ++i) o[i] *= a.so * sigma * in.from * la_pow(l2, max(i * 16 - first, 0) + 1 - a.late);
      __syncthreads();  // the scores are there

      // what the chunk's own rows give
      bool odd = false;
#pragma unroll
      for (int s = 0; s < CS; ++s) odd |= la_odd(x[s]);
      if (wave_ballot(odd)) {
        // values that are not finite must not meet the zero scores of the rows before them
#pragma unroll 1
        for (int j = C - n; j < C; ++j) {
          const typename X::Quad y = *(const typename X::Quad*)&cv[j * PV + wc + 4 * g];
#pragma unroll
          for (int i = 0; i < CT; ++i) {
            float p = 0.0f;
#pragma unroll
            for (int c = 0; c < X::FINE; ++c) p += (float)s_p[c][(i * 16 + m) * PP + X::packed(j & ~3) + (j & 3)];
            if constexpr (X::SCALED) p *= s_from[i * (i + 1) / 2 + min(j / 16, i)];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] += i * 16 + m >= j ? p * (float)y[e] : 0.0f;
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < CS; ++s)
#pragma unroll
          for (int i = 0; i < CT; ++i) {
            if (s * X::TILES > i) continue;
            Frag p[X::FINE];
#pragma unroll
            for (int c = 0; c < X::FINE; ++c) p[c] = X::packed_row(&s_p[c][(i * 16 + m) * PP + s * KB], g);
            if constexpr (X::SCALED) {  // each 16 rows' scores have a scale of their own
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (s * 2 + j <= i) {
                  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                  for (int c = 0; c < X::FINE; ++c) sum = X::mma_half(x[s], p[c], j, sum);
                  o[i] += sum * s_from[i * (i + 1) / 2 + s * 2 + j];
                }
            } else {
#pragma unroll
              for (int c = 0; c < X::FINE; ++c) o[i] = X::mma(x[s], p[c], o[i]);
            }
          }
      }
      if (WIDE) {
        if (a.out_f32)
          la_store<float, CT>((float*)out, at_o, step_o, o, first);
        else
          la_store<T, CT>((T*)out, at_o, step_o, o, first);
        out += ahead_o;
      } else {
        const int64_t to = ((a.rev ? a.T - 1 - r - m : r + m) * BH + bh) * a.DV + dv;
        if (a.out_f32)
          la_store_some<float, CT>((float*)a.out + to, a.rev ? -so : so, o, first, a.DV - dv);
        else
          la_store_some<T, CT>((T*)a.out + to, a.rev ? -so : so, o, first, a.DV - dv);
      }
    }

    since += n;
    sigma = la_pow(l2, since);
    if (!(sigma > 0x1p-16f && sigma < 0x1p16f && since < 1 << 22)) {
#pragma unroll
      for (int i = 0; i < KT; ++i) S[i] *= sigma;
      sigma = 1.0f;
      since = 0;
    }
    const float weight = __builtin_amdgcn_rcpf(sigma);
#pragma unroll
    for (int s = 0; s < CS; ++s) {
      Frag part[X::PARTS];
      float rest[KB / 4];
      unsigned big = 0;
#pragma unroll
      for (int e = 0; e < KB / 4; ++e) {
        rest[e] = (float)x[s][e] * (decay[s][e] * weight);
        big = max(big, la_bits(rest[e]));
      }
      LaScale in = {1.0f, 1.0f};
      if constexpr (X::SCALED) in = la_scale(big);
#pragma unroll
      for (int e = 0; e < KB / 4; ++e) {
        if constexpr (X::SCALED) rest[e] *= in.to;
#pragma unroll
        for (int c = 0; c < X::PARTS; ++c) {
          const L top = (L)rest[e];
          part[c][e] = top;
          rest[e] -= (float)top;
        }
      }
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const Frag y = X::col(&ck[s * KB * PK + i * 16], PK, g, m);
        if constexpr (X::SCALED) {
          f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < X::PARTS; ++c) sum = X::mma(y, part[c], sum);
          S[i] += sum * in.from;
        } else {
#pragma unroll
          for (int c = 0; c < X::PARTS; ++c) S[i] = X::mma(y, part[c], S[i]);
        }
      }
    }
    half ^= 1;
    put(half);  // zeros after the last chunk
    fetch(r + C + 2 * step <= r1 ? step : 0);
    __syncthreads();  // the next chunk is there, and the scores have been read
  }

  if (SUMS || (a.s_out && seg == a.segs - 1)) {
    float* to = a.s_out + (size_t)(SUMS ? (seg + 1) * BH + bh : bh) * size;
    asm volatile("" : "+v"(at0));  // or the first loads' addresses are held in registers up to here
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col && i * 16 + 4 * g + e < a.DK) to[at0 + (i * 16 + e) * a.sk] = sigma * S[i][e];
  }
}

// Rows of a chunk (of every type), and columns of a workgroup's block for widths DK, DV.
inline int la_chunk() { return La<float>::C; }
// 128 columns read Q and K and form the scores once where two blocks of 64 do it twice (bf16 4096 x 4 x 16
// x 128, forward and backward: 398 us, with blocks of 64 448; 4096 x 16 x 256 x 256: 377 us, with
// blocks of 64 542); 256 rows of a state in fp32 leave LDS for 64 only.
inline int la_block(int dtype, int DK, int DV) {
  return DV > 64 && (dtype != LSH_F32 || DK <= 128) ? 128 : 64;
}

// Whether the walk's rows can be read and written in whole pieces: a chunk's byte offsets stay below
// 2^30 and the output's columns come in fours.
inline bool la_wide(const LaWalk& a, int chunk) {
  const int64_t most = ((int64_t)1 << 30) / 4 / chunk;
  auto near = [&](const LaIn& x) { return x.wide && x.st >= 0 && x.st < most; };
  return near(a.q) && near(a.k) && near(a.v) && a.DV % 4 == 0 && a.B * a.H * a.DV < most;
}

// State rows that a kernel is built for, by the walk's DK.
inline int la_rows(int DK) { return DK <= 64 ? 64 : DK <= 128 ? 128 : 256; }

// Blocks of columns of the walk that has most.
inline int la_blocks(const LaWalks& all, int block) {
  int most = 0;
  for (int i = 0; i < all.n; ++i)
    if (const int n = (all.w[i].DV + block - 1) / block; n > most) most = n;
  return most;
}

// Launches walks of one la_rows and la_block (their sums: SUMS) for operands of T computed in L.
template <class T, class L>
inline int la_launch(const LaWalks& all, bool sums, hipStream_t st) {
  const LaWalk& a = all.w[0];
  const int64_t n = a.B * a.H * (sums ? a.segs - 1 : a.segs);
  if (n == 0 || all.n == 0) return LSH_OK;
  constexpr int dtype = sizeof(L) == 2 ? LSH_BF16 : LSH_F32;
  const int block = la_block(dtype, a.DK, a.DV);
  bool wide = true;
  const int blocks = la_blocks(all, block);
  for (int i = 0; i < all.n; ++i) wide = wide && la_wide(all.w[i], La<L>::C);
  if (!lm_grid_ok(n * blocks * all.n, block * 4)) return LSH_ERR_SHAPE;
  const dim3 grid((unsigned)(n * blocks * all.n));
  auto go = [&](auto dkp, auto waves) {
    constexpr int DKP = decltype(dkp)::value, W = decltype(waves)::value;
    if (sums && wide)
      k_la_walk<T, L, DKP, W, true, true><<<grid, W * 64, 0, st>>>(all);
    else if (sums)
      k_la_walk<T, L, DKP, W, true, false><<<grid, W * 64, 0, st>>>(all);
    else if (wide)
      k_la_walk<T, L, DKP, W, false, true><<<grid, W * 64, 0, st>>>(all);
    else
      k_la_walk<T, L, DKP, W, false, false><<<grid, W * 64, 0, st>>>(all);
  };
  auto with = [&](auto dkp) {
    if (block == 128)
      go(dkp, std::integral_constant<int, 8>{});
    else
      go(dkp, std::integral_constant<int, 4>{});
  };
  switch (la_rows(a.DK)) {
    case 64: with(std::integral_constant<int, 64>{}); break;
    case 128: with(std::integral_constant<int, 128>{}); break;
    default:
      if constexpr (sizeof(L) == 2)
        with(std::integral_constant<int, 256>{});
      else
        go(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
  }
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

int la_launch_f32(const LaWalks& all, bool sums, hipStream_t st);
int la_launch_bf16(const LaWalks& all, bool sums, hipStream_t st);
int la_launch_f16(const LaWalks& all, bool sums, hipStream_t st);

}  // namespace lsh
