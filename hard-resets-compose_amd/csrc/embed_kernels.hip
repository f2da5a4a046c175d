// Embedding lookup with scaling, and the table's gradient.
//
//   out[i] = scale * W[tok_i]          dW[v] = scale * sum_{i: tok_i = v} dout[i]
//
// Ids outside the table and the padding id read as zero rows and leave no gradient.  For the gradient
// the positions are sorted by token (stable, so in position order within a token) and every table row
// sums its own, in fp32 with no atomics: the same bits on every run, and every row is written once.
#include <algorithm>

#include "lsh_lm.h"

namespace lsh {

// One thread a piece of 16 bytes, or of as many columns a row's pieces apart (16384 x 1023 bf16: 12 us, with
// a thread's own columns side by side 32; 16384 x 1024 10).
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void k_embed(const int64_t* __restrict__ tok, const T* __restrict__ W,
                                               T* __restrict__ out, int64_t n, int64_t V, int D, int64_t pad,
                                               float scale, int pieces) {
  constexpr int P = kWide<T>;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t i = u / pieces;
  if (i >= n) return;
  const int d = (int)(u - i * pieces) * (WIDE ? P : 1);
  const int64_t v = tok[i];
  float f[P] = {};
  if (v >= 0 && v < V && v != pad) {
    ld_vals<P, WIDE>(f, W + (size_t)v * D, d, D, pieces);
#pragma unroll
    for (int j = 0; j < P; ++j) f[j] *= scale;
  }
  st_vals<P, WIDE>(f, out + (size_t)i * D, d, D, pieces);
}

// ---- positions by token
// The table's rows are dealt to `parts` workgroups (a power of two, row v to workgroup v % parts, so that
// frequent neighbours go to different ones); a workgroup's rows lie together in the list of positions, part
// after part.
//
// Up to kEsTile tokens one kernel does it: every workgroup reads all tokens, counts its rows' and those of
// the workgroups before it, which gives every row's place in the list, and puts its positions there in
// order.  Bound by the latency of its steps (64 tokens 9 us, 16384 uniform ones 11, with Zipf's most frequent
// token 13; many positions of few rows are put in order by all waves, which first count their shares: by one
// wave 16).
// More tokens are also split over the workgroups, or each would look at all of them: one kernel counts every
// (part, split)'s rows, the next puts its positions after those of the splits before it (65536 Zipf tokens
// 21 us, with one kernel 45; 262144 33 and about 175).
constexpr int kEsThreads = 1024, kEsPer = 16, kEsTile = kEsThreads * kEsPer, kEsWaves = kEsThreads / 64;
constexpr int kEsRuns = kEsTile / 64;
constexpr int kEsRows = 8192;  // table rows of a workgroup at most
constexpr int kEsList = 4096;  // positions on their way to the list
constexpr int kEsFew = 256, kEsFine = 512;  // more positions of at most so many rows are put by all waves

// How n tokens of V rows are dealt: splits == 0 is the one kernel.
struct EsDeal {
  int parts, splits;
  int64_t rows;  // V up to a multiple of parts
};
inline EsDeal es_deal(int64_t n, int64_t V) {
  int64_t p = n <= kEsTile ? 256 : 16;
  while ((V + p - 1) / p > kEsRows) p *= 2;
  const int splits = n <= kEsTile ? 0 : (int)std::max<int64_t>(1, std::min<int64_t>(256 / p, (n + 4095) / 4096));
  return {(int)p, splits, (int64_t)align_up((size_t)V, (size_t)p)};
}

struct EsLds {
  int row[kEsRows];              // a row's tokens, then where its next position goes
  int at[kEsList];               // positions found, in order, with
  short of[kEsList];             // the row of each
  int next[kEsWaves][kEsFine];   // the same as row for each wave's share
  int sum[kEsWaves];
  int runs[kEsRuns + 1];         // runs of 64 tokens of a tile: how many are found before each, and in all
};

// The rows of a tile's tokens, -1 for none: thread t has tokens t0 + t, t0 + t + 1024, ... before end.
__device__ __forceinline__ void es_read(int (&v)[kEsPer], const int64_t* __restrict__ tok, int t0, int end, int V,
                                        int64_t pad) {
#pragma unroll
  for (int j = 0; j < kEsPer; ++j) {
    const int i = t0 + j * kEsThreads + threadIdx.x;
    const int64_t x = i < end ? tok[i] : -1;
    v[j] = (uint64_t)x < (uint64_t)V && x != pad ? (int)x : -1;
  }
}

// The sum of a workgroup's values, in every thread.
__device__ __forceinline__ int es_sum(EsLds& s, int x) {
  x = wave_sum_i(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.sum[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0;
#pragma unroll
  for (int i = 0; i < kEsWaves; ++i) x += s.sum[i];
  __syncthreads();
  return x;
}

// Each row's place: an exclusive sum over the part's rows, 1024 at a time, behind `before` positions.  get(i,
// own): a row's positions, and how many of them lie before this workgroup's.
template <class Get>
__device__ __forceinline__ void es_places(EsLds& s, Get&& get, int rows, int before, int p, int parts, bool write,
                                          int* __restrict__ start, int* __restrict__ count) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int i0 = 0; i0 < rows; i0 += kEsThreads) {
    const int i = i0 + threadIdx.x;
    int own = 0;
    const int c = i < rows ? get(i, own) : 0;
    int incl = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(incl, o, 64);
      if (lane >= o) incl += x;
    }
    if (lane == 63) s.sum[w] = incl;
    __syncthreads();
    int at = before + incl - c;
    for (int j = 0; j < kEsWaves; ++j) {
      if (j < w) at += s.sum[j];
      before += s.sum[j];
    }
    if (i < rows) {
      s.row[i] = at + own;
      if (write) {
        start[(size_t)i * parts + p] = at;
        count[(size_t)i * parts + p] = c;
      }
    }
    __syncthreads();
  }
}

// Positions i0.. before i1 of s.at to their places by one wave, 64 at a time; next: a row's next place.
__device__ __forceinline__ void es_place(const EsLds& s, int i0, int i1, int* next, int* __restrict__ list) {
  const int lane = threadIdx.x & 63;
  const unsigned long long lower = (1ull << lane) - 1;
  for (; i0 < i1; i0 += 64) {
    const bool there = i0 + lane < i1;
    const int row = there ? s.of[i0 + lane] : -1;
    const int at = there ? s.at[i0 + lane] : 0;
    // the lanes with this lane's row
    unsigned long long same = wave_ballot(there);
    if (wave_ballot(row == __shfl(row, 0, 64)) != ~0ull) {
#pragma unroll
      for (int b = 0; b < 13; ++b) {
        const unsigned long long m = wave_ballot((row >> b) & 1);
        same &= (row >> b) & 1 ? m : ~m;
      }
    }
    if (there) {
      const int to = next[row];
      list[to + __popcll(same & lower)] = at;
      if (!(same >> lane >> 1)) next[row] = to + __popcll(same);
    }
  }
}

// The `found` positions of s.at to their places.
__device__ __forceinline__ void es_flush(EsLds& s, int found, int rows, int* __restrict__ list) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  __syncthreads();
  if (found <= kEsFew || rows > kEsFine) {
    if (w == 0) es_place(s, 0, found, s.row, list);
  } else {
    // a share for each wave, in order: what the shares before it hold of a row comes first
    const int share = (found + kEsThreads - 1) / kEsThreads * 64;
    const int i0 = min(w * share, found), i1 = min(i0 + share, found);
    for (int i = threadIdx.x; i < kEsWaves * kEsFine; i += kEsThreads) s.next[0][i] = 0;
    __syncthreads();
    for (int i = i0 + lane; i < i1; i += 64) atomicAdd(&s.next[w][s.of[i]], 1);
    __syncthreads();
    if ((int)threadIdx.x < rows) {
      int c[kEsWaves], at = s.row[threadIdx.x];
#pragma unroll
      for (int k = 0; k < kEsWaves; ++k) c[k] = s.next[k][threadIdx.x];
#pragma unroll
      for (int k = 0; k < kEsWaves; ++k) {
        s.next[k][threadIdx.x] = at;
        at += c[k];
      }
      s.row[threadIdx.x] = at;
    }
    __syncthreads();
    es_place(s, i0, i1, s.next[w], list);
  }
  __syncthreads();
}

// A tile's positions of part p to the list.
__device__ __forceinline__ void es_put(EsLds& s, const int (&v)[kEsPer], int t0, int rows, int p, int parts,
                                       int shift, int* __restrict__ list) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const unsigned long long lower = (1ull << lane) - 1;
  // where each position found goes: behind those of earlier runs of 64 tokens, then of earlier lanes
  unsigned long long hit[kEsPer];
#pragma unroll
  for (int j = 0; j < kEsPer; ++j) {
    hit[j] = wave_ballot(v[j] >= 0 && (v[j] & (parts - 1)) == p);
    if (lane == 0) s.runs[j * kEsWaves + w] = __popcll(hit[j]);
  }
  __syncthreads();
  if (w == 0) {
    constexpr int E = kEsRuns / 64;
    int c[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      c[e] = s.runs[lane * E + e];
      sum += c[e];
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(incl, o, 64);
      if (lane >= o) incl += x;
    }
    if (lane == 63) s.runs[kEsRuns] = incl;
    int at = incl - sum;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s.runs[lane * E + e] = at;
      at += c[e];
    }
  }
  __syncthreads();
  const int total = s.runs[kEsRuns];
  // the tile's positions pass through the list in windows of its size
  for (int win = 0; win < total; win += kEsList) {
#pragma unroll
    for (int j = 0; j < kEsPer; ++j) {
      const int at = s.runs[j * kEsWaves + w] + __popcll(hit[j] & lower) - win;
      if ((hit[j] >> lane & 1) && at >= 0 && at < kEsList) {
        s.at[at] = t0 + j * kEsThreads + threadIdx.x;
        s.of[at] = (short)(v[j] >> shift);
      }
    }
    es_flush(s, min(total - win, kEsList), rows, list);
  }
  __syncthreads();  // s.runs has been read
}

// n up to kEsTile.
__global__ __launch_bounds__(kEsThreads) void k_embed_sort(const int64_t* __restrict__ tok, int n, int V,
                                                           int64_t pad, int parts, int* __restrict__ start,
                                                           int* __restrict__ count, int* __restrict__ list) {
  __shared__ EsLds s;
  const int p = blockIdx.x, rows = (V - p + parts - 1) / parts, shift = __builtin_ctz(parts);
  int v[kEsPer];
  for (int i = threadIdx.x; i < rows; i += kEsThreads) s.row[i] = 0;
  __syncthreads();
  es_read(v, tok, 0, n, V, pad);
  int before = 0;
#pragma unroll
  for (int j = 0; j < kEsPer; ++j) {
    const int part = v[j] & (parts - 1);
    before += v[j] >= 0 && part < p;
    if (v[j] >= 0 && part == p) atomicAdd(&s.row[v[j] >> shift], 1);
  }
  before = es_sum(s, before);
  es_places(s, [&](int i, int&) { return s.row[i]; }, rows, before, p, parts, true, start, count);
  es_put(s, v, 0, rows, p, parts, shift, list);
}

// cnt [splits, parts, rows of a part]: the tokens of each row in each split; all [splits, parts]: their sums.
__global__ __launch_bounds__(kEsThreads) void k_embed_count(const int64_t* __restrict__ tok, int n, int V,
                                                            int64_t pad, int parts, int per, int* __restrict__ cnt,
                                                            int* __restrict__ all) {
  __shared__ EsLds s;
  const int p = blockIdx.x, rows = (V - p + parts - 1) / parts, shift = __builtin_ctz(parts);
  const int most = (V + parts - 1) / parts, t1 = (int)min((int64_t)n, (int64_t)(blockIdx.y + 1) * per);
  int v[kEsPer], mine = 0;
  for (int i = threadIdx.x; i < rows; i += kEsThreads) s.row[i] = 0;
  __syncthreads();
  for (int64_t t0 = (int64_t)blockIdx.y * per; t0 < t1; t0 += kEsTile) {
    es_read(v, tok, (int)t0, t1, V, pad);
#pragma unroll
    for (int j = 0; j < kEsPer; ++j)
      if (v[j] >= 0 && (v[j] & (parts - 1)) == p) {
        atomicAdd(&s.row[v[j] >> shift], 1);
        ++mine;
      }
  }
  mine = es_sum(s, mine);
  const size_t place = (size_t)blockIdx.y * parts + p;
  if (threadIdx.x == 0) all[place] = mine;
  for (int i = threadIdx.x; i < rows; i += kEsThreads) cnt[place * most + i] = s.row[i];
}

__global__ __launch_bounds__(kEsThreads) void k_embed_place(const int64_t* __restrict__ tok, int n, int V,
                                                            int64_t pad, int parts, int per,
                                                            const int* __restrict__ cnt, const int* __restrict__ all,
                                                            int* __restrict__ start, int* __restrict__ count,
                                                            int* __restrict__ list) {
  __shared__ EsLds s;
  const int p = blockIdx.x, rows = (V - p + parts - 1) / parts, shift = __builtin_ctz(parts);
  const int most = (V + parts - 1) / parts, splits = gridDim.y, split = blockIdx.y;
  const int t1 = (int)min((int64_t)n, (int64_t)(split + 1) * per);
  int before = 0;
  for (int i = threadIdx.x; i < splits * parts; i += kEsThreads)
    if ((i & (parts - 1)) < p) before += all[i];
  before = es_sum(s, before);
  auto get = [&](int i, int& own) {
    int c = 0;
    for (int k0 = 0; k0 < splits; k0 += 8) {
      int x[8];  // the loads first
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = cnt[((size_t)min(k0 + k, splits - 1) * parts + p) * most + i];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] = k0 + k < splits ? x[k] : 0;
        c += x[k];
        own += k0 + k < split ? x[k] : 0;
      }
    }
    return c;
  };
  es_places(s, get, rows, before, p, parts, split == 0, start, count);
  for (int64_t t0 = (int64_t)split * per; t0 < t1; t0 += kEsTile) {
    int v[kEsPer];
    es_read(v, tok, (int)t0, t1, V, pad);
    es_put(s, v, (int)t0, rows, p, parts, shift, list);
  }
}

// A workgroup takes a block of kEbLanes*16 bytes of columns; a table row is taken by `lanes` lanes of a
// wave, 16 bytes a lane, so a wave takes 4 rows or more at once.  Up to kEbFew positions are summed by the
// row's own lanes; longer rows are dealt to the workgroup's waves, up to kEbHot positions to one (its lane
// groups take positions in turn), more to all, always joined in a fixed order.  Neighbouring rows, which
// are often frequent together, go to different workgroups.
// Bound by the rows read and written (16384 tokens, 32000 x 1024 bf16: 97 MB, 26 us; 262144 uniform tokens 600
// MB, 156 us) and, with a Zipf text, by its most frequent token, whose rows one workgroup sums for a block of
// columns (262144 tokens: 213 us).  8 waves and 4 groups a wave measured best: with the sort 40 us; 16 waves
// took 8 us more, 4 waves 6.  Blocks of 512 and 1024 bytes take 31 and 30 us with uniform tokens where 256
// take 33, but 41 and 48 with Zipf's where 256 take 39.  Rows of 1023 columns, element by element: 65 us.
constexpr int kEbThreads = 512, kEbLanes = 16, kEbFew = 4, kEbHot = 256, kEbGroups = 32;

// The sum of dout's rows at list[begin .. begin + n) in columns d.., dealt to `groups` lane groups, this
// lane's the group-th, Q positions at once.
template <class T, bool WIDE, int Q, class At>
__device__ __forceinline__ void eb_sum(float (&t)[kWide<T>], At&& at, int n, int group, int groups,
                                       const T* __restrict__ dout, int d, int D, int lanes) {
  constexpr int P = kWide<T>;
  for (int i = group; i < n; i += Q * groups) {
    Raw<P, WIDE, T> x[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) x[q].load(dout + (size_t)at(min(i + q * groups, n - 1)) * D, d, D, lanes);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float f[P];
      x[q].get(f, d, D, lanes, i + q * groups < n);
#pragma unroll
      for (int j = 0; j < P; ++j) t[j] += f[j];
    }
  }
}

template <class T, bool WIDE>
__global__ __launch_bounds__(kEbThreads) void k_embed_bwd(const int* __restrict__ start,
                                                          const int* __restrict__ count,
                                                          const int* __restrict__ list,
                                                          const T* __restrict__ dout, T* __restrict__ dW, int n,
                                                          int V, int D, float scale, int lanes) {
  constexpr int P = kWide<T>, WAVES = kEbThreads / 64, EACH = kEbGroups / WAVES;
  // longer rows with their places and lengths, from the front; the longest from the back
  __shared__ int s_row[kEbGroups * 64], s_begin[kEbGroups * 64], s_count[kEbGroups * 64], s_n[2];
  __shared__ int s_list[WAVES * kEbHot];
  __shared__ float s_sum[WAVES][kEbLanes * P];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int per = 64 / lanes, sub = lane / lanes, l = lane % lanes;  // rows of a wave, this lane's, its place
  const int d0 = blockIdx.y * kEbLanes * P, d = d0 + (WIDE ? l * P : l);
  if (threadIdx.x < 2) s_n[threadIdx.x] = 0;
  __syncthreads();
  int c[EACH], at[EACH][kEbFew];
  bool any[EACH];  // whether a row of the wave has positions
  int64_t row[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    // short rows stay with their neighbours, so that a wave writes whole lines
    const int g = k * WAVES + w;
    row[k] = lanes == kEbLanes ? (int64_t)(g * per + sub) * gridDim.x + blockIdx.x
                               : ((int64_t)g * gridDim.x + blockIdx.x) * per + sub;
    c[k] = row[k] < V ? count[row[k]] : -1;
    at[k][0] = row[k] < V ? start[row[k]] : 0;
  }
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    if (c[k] > kEbFew) {
      if (l == 0) {
        const bool hot = c[k] > kEbHot;
        const int i = atomicAdd(&s_n[hot], 1), to = hot ? kEbGroups * 64 - 1 - i : i;
        s_row[to] = (int)row[k], s_begin[to] = at[k][0], s_count[to] = c[k];
      }
      c[k] = -1;
    }
    any[k] = wave_ballot(c[k] > 0) != 0;
    if (any[k])
#pragma unroll
      for (int q = kEbFew - 1; q >= 0; --q) at[k][q] = n > 0 ? list[min(at[k][0] + q, n - 1)] : 0;
  }
  Raw<P, WIDE, T> x[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k)
    if (any[k]) x[k].load(dout + (size_t)(c[k] > 0 ? at[k][0] : 0) * D, d, D, lanes);
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    float s[P] = {};
    if (any[k]) {
      x[k].get(s, d, D, lanes, c[k] > 0);
      if (wave_ballot(c[k] > 1)) {
        Raw<P, WIDE, T> y[kEbFew - 1];
#pragma unroll
        for (int q = 1; q < kEbFew; ++q) y[q - 1].load(dout + (size_t)(q < c[k] ? at[k][q] : 0) * D, d, D, lanes);
#pragma unroll
        for (int q = 1; q < kEbFew; ++q) {
          float f[P];
          y[q - 1].get(f, d, D, lanes, q < c[k]);
#pragma unroll
          for (int j = 0; j < P; ++j) s[j] += f[j];
        }
      }
    }
    if (c[k] < 0) continue;
#pragma unroll
    for (int j = 0; j < P; ++j) s[j] *= scale;
    st_vals<P, WIDE>(s, dW + (size_t)row[k] * D, d, D, lanes);
  }
  __syncthreads();
  for (int h = w; h < s_n[0]; h += WAVES) {
    const int v = s_row[h], n = s_count[h], begin = s_begin[h];
    int* mine = s_list + w * kEbHot;
    for (int i = lane; i < n; i += 64) mine[i] = list[begin + i];
    __builtin_amdgcn_wave_barrier();
    float t[P] = {};
    eb_sum<T, WIDE, 8>(t, [&](int i) { return mine[i]; }, n, sub, per, dout, d, D, lanes);
    for (int o = lanes; o < 64; o *= 2)
#pragma unroll
      for (int j = 0; j < P; ++j) t[j] += __shfl_xor(t[j], o, 64);
    if (sub == 0) {
#pragma unroll
      for (int j = 0; j < P; ++j) t[j] *= scale;
      st_vals<P, WIDE>(t, dW + (size_t)v * D, d, D, lanes);
    }
    __builtin_amdgcn_wave_barrier();
  }
  for (int h = kEbGroups * 64 - s_n[1]; h < kEbGroups * 64; ++h) {
    const int v = s_row[h], n = s_count[h], begin = s_begin[h];
    float t[P] = {};
    for (int i0 = 0; i0 < n; i0 += WAVES * kEbHot) {
      const int m = min(n - i0, WAVES * kEbHot);
      __syncthreads();  // s_list and s_sum have been read
      for (int i = threadIdx.x; i < m; i += kEbThreads) s_list[i] = list[begin + i0 + i];
      __syncthreads();
      eb_sum<T, WIDE, 8>(t, [&](int i) { return s_list[i]; }, m, w * per + sub, per * WAVES, dout, d, D, lanes);
    }
    for (int o = lanes; o < 64; o *= 2)
#pragma unroll
      for (int j = 0; j < P; ++j) t[j] += __shfl_xor(t[j], o, 64);
    if (sub == 0)
#pragma unroll
      for (int j = 0; j < P; ++j) s_sum[w][l * P + j] = t[j];
    __syncthreads();
    if ((int)threadIdx.x < lanes) {
#pragma unroll
      for (int j = 0; j < P; ++j) t[j] = 0.0f;
      for (int k = 0; k < WAVES; ++k)
#pragma unroll
        for (int j = 0; j < P; ++j) t[j] += s_sum[k][threadIdx.x * P + j];
#pragma unroll
      for (int j = 0; j < P; ++j) t[j] *= scale;
      st_vals<P, WIDE>(t, dW + (size_t)v * D, d, D, lanes);
    }
  }
}

static int embed_check(int dtype, int64_t n, int64_t V, int64_t D) {
  if (!lm_dtype_ok(dtype)) return LSH_ERR_ARG;
  if (n < 0 || n > 0x7fffffff - kEsTile || V < 0 || V > 0x7fffffff / 2 || D < 1 || D > (1 << 18))
    return LSH_ERR_SHAPE;
  return LSH_OK;
}

// Whether rows of D elements of a type begin at multiples of 16 bytes in both arrays.
static bool embed_wide(int dtype, int64_t D, const void* a, const void* b) {
  return D * lm_dtype_size(dtype) % 16 == 0 && (uintptr_t)a % 16 == 0 && (uintptr_t)b % 16 == 0;
}

}  // namespace lsh

using namespace lsh;

extern "C" int lsh_embed_fwd(int dtype, const int64_t* tokens, const void* weight, void* out, int64_t n,
                             int64_t V, int64_t D, int64_t padding, float scale, void* stream) {
  if (int rc = embed_check(dtype, n, V, D)) return rc;
  if (n == 0) return LSH_OK;
  if (bad_ptr(tokens) || (V > 0 && bad_ptr(weight)) || bad_ptr(out)) return LSH_ERR_ARG;
  const int per = 16 / lm_dtype_size(dtype), pieces = (int)((D + per - 1) / per);
  const int64_t blocks = (n * pieces + 255) / 256;
  if (!lm_grid_ok(blocks, 256)) return LSH_ERR_SHAPE;
  const bool wide = embed_wide(dtype, D, weight, out);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel) {
      kernel<<<dim3((unsigned)blocks), 256, 0, (hipStream_t)stream>>>(tokens, (const T*)weight, (T*)out, n, V,
                                                                     (int)D, padding, scale, pieces);
    };
    if (wide)
      go(k_embed<T, true>);
    else
      go(k_embed<T, false>);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}

extern "C" size_t lsh_embed_bwd_workspace(int64_t n, int64_t V) {
  if (embed_check(LSH_F32, n, V, 1)) return 0;
  const EsDeal d = es_deal(n, V);
  return (size_t)(2 * d.rows + n + d.splits * (d.rows + d.parts)) * sizeof(int);
}

extern "C" int lsh_embed_bwd(int dtype, const int64_t* tokens, const void* dout, void* dweight, int64_t n,
                             int64_t V, int64_t D, int64_t padding, float scale, void* ws, size_t ws_bytes,
                             void* stream) {
  if (int rc = embed_check(dtype, n, V, D)) return rc;
  if (V == 0) return LSH_OK;
  if (bad_ptr(dweight) || (n > 0 && (bad_ptr(tokens) || bad_ptr(dout)))) return LSH_ERR_ARG;
  if (bad_ptr(ws) || ws_bytes < lsh_embed_bwd_workspace(n, V)) return LSH_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const EsDeal d = es_deal(n, V);
  int *start = (int*)ws, *count = start + d.rows, *list = count + d.rows;
  if (d.splits == 0) {
    k_embed_sort<<<dim3((unsigned)d.parts), kEsThreads, 0, st>>>(tokens, (int)n, (int)V, padding, d.parts, start,
                                                                count, list);
  } else {
    const int share = (int)((n + d.splits - 1) / d.splits);
    const dim3 grid((unsigned)d.parts, (unsigned)d.splits);
    int *all = list + n, *cnt = all + (size_t)d.splits * d.parts;
    k_embed_count<<<grid, kEsThreads, 0, st>>>(tokens, (int)n, (int)V, padding, d.parts, share, cnt, all);
    LSH_CHECK_LAUNCH();
    k_embed_place<<<grid, kEsThreads, 0, st>>>(tokens, (int)n, (int)V, padding, d.parts, share, cnt, all, start,
                                              count, list);
  }
  LSH_CHECK_LAUNCH();
  const int per = 16 / lm_dtype_size(dtype);
  int lanes = 1;
  while (lanes < kEbLanes && lanes * per < D) lanes *= 2;
  const int64_t groups = (V + 64 / lanes - 1) / (64 / lanes);
  const dim3 grid((unsigned)((groups + kEbGroups - 1) / kEbGroups), (unsigned)((D + kEbLanes * per - 1) / (kEbLanes * per)));
  const bool wide = embed_wide(dtype, D, dout, dweight);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel) {
      kernel<<<grid, kEbThreads, 0, st>>>(start, count, list, (const T*)dout, (T*)dweight, (int)n, (int)V, (int)D,
                                          scale, lanes);
    };
    if (wide)
      go(k_embed_bwd<T, true>);
    else
      go(k_embed_bwd<T, false>);
  });
  LSH_CHECK_LAUNCH();
  return LSH_OK;
}
