// Attention of every node over its neighbours: the softmax of each row of a CSR
// pattern, forward and backward.
//
//   s(i,j) = scale * <q_i, k_j> + value(i,j)          j in row i, edge kept
//   out_i  = sum_j p(i,j) v_j,   p(i,j) = exp(s(i,j) - m_i) * r_i,
//   m_i = max_j s(i,j),          r_i = 1 / sum_j exp(s(i,j) - m_i)
//
// Backward, the probabilities formed again from the two numbers m_i, r_i kept per
// row and head (nothing of the size of the pattern is stored):
//
//   delta_i = <dout_i, out_i>       ds(i,j) = p(i,j) * (<dout_i, v_j> - delta_i)
//   dq_i = scale * sum_j ds k_j     dk_j = scale * sum_i ds q_i     dv_j = sum_i p dout_i
//
// dq is a pass over the rows of the pattern, dk / dv one over the rows of its
// transpose: every sum has one owner and a fixed order, so there are no atomics and
// results are the same bits run to run.
//
// m and r are kept instead of the one number m - log r: at logits of 10^4, or a row
// whose every value is the type's lowest, fp32 has no digits left for log r.
#include "gcnx_common.h"

namespace gcnx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// A lane's piece of one head's vector: 16 bytes.
template <typename T> struct Piece;
template <> struct Piece<float> { typedef f32x4 raw; static constexpr int N = 4; };
template <> struct Piece<__bf16> { typedef bf16x8 raw; static constexpr int N = 8; };
template <> struct Piece<_Float16> { typedef f16x8 raw; static constexpr int N = 8; };

// `n` elements at p (n <= 0: none) into the piece, zeros behind them.  WIDE: p is
// 16-byte aligned and n is either >= the piece or <= 0.
template <typename T, bool WIDE>
__device__ __forceinline__ typename Piece<T>::raw load_piece(const T *p, int n) {
  typename Piece<T>::raw x = {};
  if constexpr (WIDE) {
    if (n > 0) x = *reinterpret_cast<const typename Piece<T>::raw *>(p);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i)
      if (i < n) x[i] = p[i];
  }
  return x;
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store_piece(T *p, int n, const float (&v)[Piece<T>::N]) {
  if constexpr (WIDE) {
    if (n > 0) {
      typename Piece<T>::raw x;
#pragma unroll
      for (int i = 0; i < Piece<T>::N; ++i) x[i] = (T)v[i];
      *reinterpret_cast<typename Piece<T>::raw *>(p) = x;
    }
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

// Sum over groups of G neighbouring lanes, the result in every lane of the group.
// Steps 1..8 are moves on the vector ALU: quad permutes, then the mirrors of 8 and
// 16 lanes (every lane of a sub-group already holds the sub-group's sum).
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#define GCNX_DPP(ctrl) __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), ctrl, 0xF, 0xF, true))
  if constexpr (G >= 2) v += GCNX_DPP(0xB1);
  if constexpr (G >= 4) v += GCNX_DPP(0x4E);
  if constexpr (G >= 8) v += GCNX_DPP(0x141);
  if constexpr (G >= 16) v += GCNX_DPP(0x140);
  if constexpr (G >= 32) v += __shfl_xor(v, 16, kWave);
  if constexpr (G >= 64) v += __shfl_xor(v, 32, kWave);
#undef GCNX_DPP
  return v;
}

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
__device__ __forceinline__ bool is_lowest(float x) { return x == -__builtin_inff(); }

// Rows longer than this are cut at the multiples of it in the order of the
// nonzeros, a wavefront per piece, and joined by a second kernel.
constexpr int kSegment = 512;
constexpr int kUnroll = 4;   // edges in flight per lane

struct AttnArgs {
  // pattern walked by this pass (the matrix, or its transpose)
  const int64_t *row_ptr;
  const int32_t *col_idx;
  const float *val;             // NULL: no logit shifts
  const uint8_t *mask;          // NULL: every edge stays
  const int64_t *mask_index;    // NULL: in the order of the nonzeros
  const int32_t *chunk_row;
  int64_t n_rows, nnz;
  // operands; strides in elements
  const void *q, *k, *v, *out, *dout;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head, dout_row, dout_head;
  int32_t heads, kv_heads, group, dim;
  float scale;
  // results
  void *o0, *o1;
  int64_t o0_row, o0_head, o1_row, o1_head;
  float *stats;                 // forward: 2 per row and head; backward row pass reads them
  f32x4 *stats4;                // backward: m, r, delta per row and head
  // work split
  float *part;                  // partial results of cut rows
  int64_t part_floats;          // per piece
  int64_t n_pieces;             // 2 * chunks of kSegment nonzeros, 0: no row is cut
  int32_t slot_heads_log2;      // heads side by side in a wavefront
  int32_t edge_log2, row_log2;  // edges of a row, rows side by side in a wavefront
};

// What one group of lanes works on.
struct Task {
  int64_t row, beg, end;
  int64_t piece;                // >= 0: a piece of a cut row
  bool write;
  int32_t edge, edges;          // this lane's place among the edges side by side
  int32_t head, d0, n;          // head, first element and elements of the lane's piece
};

template <typename T, int LPH>
__device__ __forceinline__ bool find_task(const AttnArgs &p, int heads, Task &t) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t task = (int64_t)blockIdx.x * kWavesPerBlock + (threadIdx.x >> 6);
  const int piece = lane % LPH, slot = lane / LPH;
  const int hs = slot & ((1 << p.slot_heads_log2) - 1);
  int rest = slot >> p.slot_heads_log2;
  t.head = ((int)blockIdx.y << p.slot_heads_log2) + hs;
  t.d0 = piece * Piece<T>::N;
  t.n = t.head < heads ? p.dim - t.d0 : 0;
  if (task < p.n_pieces) {
    t.edge = rest;
    t.edges = (kWave / LPH) >> p.slot_heads_log2;
    const int64_t first = (task >> 1) * kSegment, next = first + kSegment;
    if (task & 1) {             // the cut row that begins in this chunk
      if (next >= p.nnz) return false;
      t.row = p.chunk_row[next / kChunkUnit];
      t.beg = p.row_ptr[t.row];
      t.end = p.row_ptr[t.row + 1];
      if (t.beg < first || t.beg >= next || t.end - t.beg <= kSegment) return false;
      t.end = next;
    } else {                    // the cut row that goes on into this chunk
      t.row = p.chunk_row[first / kChunkUnit];
      t.beg = p.row_ptr[t.row];
      t.end = p.row_ptr[t.row + 1];
      if (t.beg >= first || t.end - t.beg <= kSegment) return false;
      t.beg = first;
      t.end = t.end < next ? t.end : next;
    }
    t.piece = task;
    t.write = true;
  } else {
    t.edge = rest & ((1 << p.edge_log2) - 1);
    t.edges = 1 << p.edge_log2;
    t.row = ((task - p.n_pieces) << p.row_log2) + (rest >> p.edge_log2);
    t.piece = -1;
    t.write = t.row < p.n_rows;
    t.beg = t.write ? p.row_ptr[t.row] : 0;
    t.end = t.write ? p.row_ptr[t.row + 1] : 0;
    if (p.n_pieces && t.end - t.beg > kSegment) {
      t.write = false;
      t.end = t.beg;
    }
  }
  return true;
}

// One edge: its column, its logit shift, whether it takes part.  An edge whose
// shift is -inf is out of the softmax like a masked one: its operands are not read,
// so infinities and NaN in masked places stay where they are.
__device__ __forceinline__ bool load_edge(const AttnArgs &p, int64_t e, int64_t end, int32_t &col, float &shift) {
  col = 0;
  shift = 0.0f;
  bool on = e < end;
  if (on) {
    col = p.col_idx[e];
    if (p.val) {
      shift = p.val[e];
      on = !is_lowest(shift);
    }
    if (p.mask) on = on && p.mask[p.mask_index ? p.mask_index[e] : e] != 0;
  }
  return on;
}

template <typename T>
__device__ __forceinline__ void widen(const typename Piece<T>::raw &x, float (&f)[Piece<T>::N]) {
#pragma unroll
  for (int i = 0; i < Piece<T>::N; ++i) f[i] = (float)x[i];
}

// Joins two softmax states (m, l, acc); m = -inf: nothing summed yet.
template <int N>
__device__ __forceinline__ void join(float &m, float &l, float (&acc)[N], float m2, float l2, const float (&acc2)[N]) {
  const float top = fmaxf(m, m2), safe = is_lowest(top) ? 0.0f : top;
  const float a = exp_of(m - safe), b = exp_of(m2 - safe);
  m = top;
  l = l * a + l2 * b;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = acc[i] * a + acc2[i] * b;
}

template <typename T, bool WIDE, int N>
__device__ __forceinline__ void finish_forward(const AttnArgs &p, const Task &t, float m, float l, const float (&acc)[N]) {
  const float r = l == 0.0f ? 0.0f : 1.0f / l;      // nothing takes part: zeros
  float o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = acc[i] * r;
  store_piece<T, WIDE>((T *)p.o0 + t.row * p.o0_row + t.head * p.o0_head + t.d0, t.n, o);
  if (p.stats && t.d0 == 0 && t.n > 0) {
    float *st = p.stats + (t.row * p.heads + t.head) * 2;
    st[0] = is_lowest(m) ? 0.0f : m;
    st[1] = r;
  }
}

template <typename T, int LPH, bool WIDE>
__global__ __launch_bounds__(kBlock) void attention_forward_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N;
  Task t;
  if (!find_task<T, LPH>(p, p.heads, t)) return;
  const int kv = t.head / p.group;
  float q[N], acc[N] = {};
  widen<T>(load_piece<T, WIDE>((const T *)p.q + t.row * p.q_row + t.head * p.q_head + t.d0, t.write ? t.n : 0), q);
  const T *kb = (const T *)p.k + kv * p.k_head + t.d0, *vb = (const T *)p.v + kv * p.v_head + t.d0;
  float m = -__builtin_inff(), l = 0.0f;
  for (int64_t e = t.beg + t.edge; e < t.end; e += kUnroll * t.edges) {
    int32_t col[kUnroll];
    float s[kUnroll];
    bool on[kUnroll];
    typename Piece<T>::raw k[kUnroll], v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) on[u] = load_edge(p, e + u * t.edges, t.end, col[u], s[u]);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      k[u] = load_piece<T, WIDE>(kb + col[u] * p.k_row, on[u] ? t.n : 0);
      v[u] = load_piece<T, WIDE>(vb + col[u] * p.v_row, on[u] ? t.n : 0);
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float d = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) d = fmaf(q[i], (float)k[u][i], d);
      d = group_sum<LPH>(d);
      s[u] = on[u] ? fmaf(d, p.scale, s[u]) : -__builtin_inff();
      top = fmaxf(top, s[u]);
    }
    const float safe = is_lowest(top) ? 0.0f : top;
    const float keep = exp_of(m - safe);
    m = top;
    l *= keep;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= keep;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const float w = exp_of(s[u] - safe);
      l += w;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = fmaf(w, (float)v[u][i], acc[i]);
    }
  }
  for (int at = 1; at < t.edges; at <<= 1) {
    const int off = (LPH * at) << p.slot_heads_log2;
    float m2 = __shfl_xor(m, off, kWave), l2 = __shfl_xor(l, off, kWave), acc2[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc2[i] = __shfl_xor(acc[i], off, kWave);
    join<N>(m, l, acc, m2, l2, acc2);
  }
  if (t.edge != 0 || !t.write || t.n <= 0) return;
  if (t.piece >= 0) {
    float *part = p.part + t.piece * p.part_floats + (int64_t)t.head * (LPH * N + 2);
#pragma unroll
    for (int i = 0; i < N; ++i) part[2 + t.d0 + i] = acc[i];
    if (t.d0 == 0) {
      part[0] = m;
      part[1] = l;
    }
    return;
  }
  finish_forward<T, WIDE>(p, t, m, l, acc);
}

// The cut row that begins in chunk blockIdx.x, if there is one: its pieces are
// slot 1 of that chunk and slot 0 of the chunks after it.
__device__ __forceinline__ bool find_cut_row(const AttnArgs &p, int64_t &row, int64_t &last) {
  const int64_t first = (int64_t)blockIdx.x * kSegment, next = first + kSegment;
  if (next >= p.nnz) return false;
  row = p.chunk_row[next / kChunkUnit];
  const int64_t beg = p.row_ptr[row], end = p.row_ptr[row + 1];
  if (beg < first || beg >= next || end - beg <= kSegment) return false;
  last = (end - 1) / kSegment;
  return true;
}

// Joins the pieces of cut rows.  A workgroup per row and head tile: the pieces are
// dealt to the lane groups, each joins its own in order, then the groups are joined
// through LDS in order: a fixed tree.
template <typename T, int LPH, bool WIDE>
__global__ __launch_bounds__(kBlock) void attention_forward_join_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N;
  __shared__ float sh[kBlock][N + 2];
  Task t;
  int64_t last;
  if (!find_cut_row(p, t.row, last)) return;
  const int lane = threadIdx.x & (kWave - 1);
  const int piece = lane % LPH, slot = lane / LPH, hs = slot & ((1 << p.slot_heads_log2) - 1);
  const int per_wave = (kWave / LPH) >> p.slot_heads_log2, groups = per_wave * kWavesPerBlock;
  const int group = (slot >> p.slot_heads_log2) + per_wave * (threadIdx.x >> 6);
  t.head = ((int)blockIdx.y << p.slot_heads_log2) + hs;
  t.d0 = piece * N;
  t.n = t.head < p.heads ? p.dim - t.d0 : 0;
  float m = -__builtin_inff(), l = 0.0f, acc[N] = {};
  if (t.n > 0)
    for (int64_t c = blockIdx.x + group; c <= last; c += groups) {
      const float *part = p.part + (c * 2 + (c == blockIdx.x)) * p.part_floats + (int64_t)t.head * (LPH * N + 2);
      float a2[N];
#pragma unroll
      for (int i = 0; i < N; ++i) a2[i] = part[2 + t.d0 + i];
      join<N>(m, l, acc, part[0], part[1], a2);
    }
  float *mine = sh[threadIdx.x];
  mine[0] = m;
  mine[1] = l;
#pragma unroll
  for (int i = 0; i < N; ++i) mine[2 + i] = acc[i];
  __syncthreads();
  if (group != 0 || t.n <= 0) return;
  for (int g = 1; g < groups; ++g) {
    const float *other = sh[(g / per_wave) * kWave + (((g % per_wave) << p.slot_heads_log2) + hs) * LPH + piece];
    float a2[N];
#pragma unroll
    for (int i = 0; i < N; ++i) a2[i] = other[2 + i];
    join<N>(m, l, acc, other[0], other[1], a2);
  }
  finish_forward<T, WIDE>(p, t, m, l, acc);
}

// Row pass of the backward: delta, dq.  Writes m, r, delta side by side for the
// column pass.
//
// delta from the stored output carries that output's rounding, which in 16 bits is
// larger than the differences <dout, v_j> - delta of a row whose values are alike.
// So <dout, out> is only a first value d0; the pass sums what it is off by,
//   rest = sum_j p (<dout, v_j> - d0),   and beside  A = sum_j p (<dout, v_j> - d0) k_j
// also B = sum_j p k_j:  delta = d0 + rest,  dq = scale (A - rest B).
template <typename T>
constexpr bool kCorrected = sizeof(T) == 2;

template <typename T, bool WIDE, int N>
__device__ __forceinline__ void finish_rows(const AttnArgs &p, const Task &t, float m, float r, float d0, float rest,
                                            float (&a)[N], const float (&b)[N]) {
  if (t.d0 == 0) p.stats4[t.row * p.heads + t.head] = f32x4{m, r, d0 + rest, 0.0f};
  if (!p.o0) return;
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = (kCorrected<T> ? fmaf(-rest, b[i], a[i]) : a[i]) * p.scale;
  store_piece<T, WIDE>((T *)p.o0 + t.row * p.o0_row + t.head * p.o0_head + t.d0, t.n, a);
}

// What a row's lanes hold of it in the row pass.
template <typename T, int LPH, bool WIDE>
__device__ __forceinline__ void load_row(const AttnArgs &p, const Task &t, float (&g)[Piece<T>::N], float &m, float &r, float &d0) {
  constexpr int N = Piece<T>::N;
  const int n = t.write ? t.n : 0;
  float o[N];
  widen<T>(load_piece<T, WIDE>((const T *)p.dout + t.row * p.dout_row + t.head * p.dout_head + t.d0, n), g);
  widen<T>(load_piece<T, WIDE>((const T *)p.out + t.row * p.out_row + t.head * p.out_head + t.d0, n), o);
  d0 = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) d0 = fmaf(g[i], o[i], d0);
  d0 = group_sum<LPH>(d0);
  m = r = 0.0f;
  if (t.write && t.head < p.heads) {
    const float *st = p.stats + (t.row * p.heads + t.head) * 2;
    m = st[0];
    r = st[1];
  }
  if (r == 0.0f) d0 = 0.0f;     // a row of zeros hands nothing on, whatever its gradient holds
}

template <typename T, int LPH, bool WIDE>
__global__ __launch_bounds__(kBlock) void attention_backward_rows_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N;
  Task t;
  if (!find_task<T, LPH>(p, p.heads, t)) return;
  const int kv = t.head / p.group;
  float q[N], g[N], acc[N] = {}, low[N] = {}, m, r, d0, rest = 0.0f;
  widen<T>(load_piece<T, WIDE>((const T *)p.q + t.row * p.q_row + t.head * p.q_head + t.d0, t.write ? t.n : 0), q);
  load_row<T, LPH, WIDE>(p, t, g, m, r, d0);
  const T *kb = (const T *)p.k + kv * p.k_head + t.d0, *vb = (const T *)p.v + kv * p.v_head + t.d0;
  if (!kCorrected<T> && !p.o0) t.end = t.beg;      // delta alone is asked for
  for (int64_t e = t.beg + t.edge; e < t.end; e += kUnroll * t.edges) {
    int32_t col[kUnroll];
    float shift[kUnroll];
    bool on[kUnroll];
    typename Piece<T>::raw k[kUnroll], v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) on[u] = load_edge(p, e + u * t.edges, t.end, col[u], shift[u]);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      k[u] = load_piece<T, WIDE>(kb + col[u] * p.k_row, on[u] ? t.n : 0);
      v[u] = load_piece<T, WIDE>(vb + col[u] * p.v_row, on[u] ? t.n : 0);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float s = 0.0f, d = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s = fmaf(q[i], (float)k[u][i], s);
        d = fmaf(g[i], (float)v[u][i], d);
      }
      s = group_sum<LPH>(s);
      d = group_sum<LPH>(d);
      const float w = on[u] ? exp_of(fmaf(s, p.scale, shift[u]) - m) * r : 0.0f;
      const float ds = on[u] ? w * (d - d0) : 0.0f;
      rest += ds;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        acc[i] = fmaf(ds, (float)k[u][i], acc[i]);
        if constexpr (kCorrected<T>) low[i] = fmaf(w, (float)k[u][i], low[i]);
      }
    }
  }
  for (int at = 1; at < t.edges; at <<= 1) {
    const int off = (LPH * at) << p.slot_heads_log2;
    rest += __shfl_xor(rest, off, kWave);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      acc[i] += __shfl_xor(acc[i], off, kWave);
      if constexpr (kCorrected<T>) low[i] += __shfl_xor(low[i], off, kWave);
    }
  }
  if (!kCorrected<T>) rest = 0.0f;
  if (t.edge != 0 || !t.write || t.n <= 0) return;
  if (t.piece >= 0) {
    float *part = p.part + t.piece * p.part_floats + (int64_t)t.head * (2 * LPH * N + 1);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      part[t.d0 + i] = acc[i];
      part[LPH * N + t.d0 + i] = low[i];
    }
    if (t.d0 == 0) part[2 * LPH * N] = rest;
    return;
  }
  finish_rows<T, WIDE>(p, t, m, r, d0, rest, acc, low);
}

// Column pass: a row of the transpose is a column j of the pattern.  The lanes own
// the key heads; the edges of the column are walked once per query head that
// shares the key head, as edges * group items.
template <typename T, int LPH, bool WIDE>
__global__ __launch_bounds__(kBlock) void attention_backward_columns_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N;
  Task t;
  if (!find_task<T, LPH>(p, p.kv_heads, t)) return;
  const int n_row = t.write ? t.n : 0;
  float k[N], v[N], dk[N] = {}, dv[N] = {};
  widen<T>(load_piece<T, WIDE>((const T *)p.k + t.row * p.k_row + t.head * p.k_head + t.d0, n_row), k);
  widen<T>(load_piece<T, WIDE>((const T *)p.v + t.row * p.v_row + t.head * p.v_head + t.d0, n_row), v);
  const T *qb = (const T *)p.q + t.d0, *gb = (const T *)p.dout + t.d0;
  const int64_t items = (t.end - t.beg) * p.group;
  for (int64_t it = t.edge; it < items; it += kUnroll * t.edges) {
    int32_t row[kUnroll], head[kUnroll];
    float shift[kUnroll];
    bool on[kUnroll];
    typename Piece<T>::raw q[kUnroll], g[kUnroll];
    f32x4 st[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t x = it + u * t.edges;
      const int64_t e = p.group == 1 ? x : items <= 0xffffffffll ? (int64_t)((uint32_t)x / (uint32_t)p.group) : x / p.group;
      head[u] = t.head * p.group + (int)(x - e * p.group);
      on[u] = load_edge(p, t.beg + e, t.end, row[u], shift[u]) && t.n > 0;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      q[u] = load_piece<T, WIDE>(qb + row[u] * p.q_row + head[u] * p.q_head, on[u] ? t.n : 0);
      g[u] = load_piece<T, WIDE>(gb + row[u] * p.dout_row + head[u] * p.dout_head, on[u] ? t.n : 0);
      st[u] = on[u] ? p.stats4[(int64_t)row[u] * p.heads + head[u]] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float s = 0.0f, d = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s = fmaf(k[i], (float)q[u][i], s);
        d = fmaf(v[i], (float)g[u][i], d);
      }
      s = group_sum<LPH>(s);
      d = group_sum<LPH>(d);
      const float w = on[u] ? exp_of(fmaf(s, p.scale, shift[u]) - st[u][0]) * st[u][1] : 0.0f;
      const float ds = on[u] ? w * (d - st[u][2]) : 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        dv[i] = fmaf(w, (float)g[u][i], dv[i]);
        dk[i] = fmaf(ds, (float)q[u][i], dk[i]);
      }
    }
  }
  for (int at = 1; at < t.edges; at <<= 1) {
    const int off = (LPH * at) << p.slot_heads_log2;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      dk[i] += __shfl_xor(dk[i], off, kWave);
      dv[i] += __shfl_xor(dv[i], off, kWave);
    }
  }
  if (t.edge != 0 || !t.write || t.n <= 0) return;
  if (t.piece >= 0) {
    float *part = p.part + t.piece * p.part_floats + (int64_t)t.head * (2 * LPH * N + 1);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      part[t.d0 + i] = dk[i];
      part[LPH * N + t.d0 + i] = dv[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) dk[i] *= p.scale;
  store_piece<T, WIDE>((T *)p.o0 + t.row * p.o0_row + t.head * p.o0_head + t.d0, t.n, dk);
  store_piece<T, WIDE>((T *)p.o1 + t.row * p.o1_row + t.head * p.o1_head + t.d0, t.n, dv);
}

// Adds the pieces of cut rows in the backward passes: two vectors and a number a
// head (A, B and rest of the row pass; dk, dv and nothing of the column pass).
template <typename T, int LPH, bool WIDE, bool COLUMNS>
__global__ __launch_bounds__(kBlock) void attention_backward_join_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N;
  __shared__ float sh[kBlock][2 * N + 1];
  Task t;
  int64_t last;
  if (!find_cut_row(p, t.row, last)) return;
  const int heads = COLUMNS ? p.kv_heads : p.heads;
  const int lane = threadIdx.x & (kWave - 1);
  const int piece = lane % LPH, slot = lane / LPH, hs = slot & ((1 << p.slot_heads_log2) - 1);
  const int per_wave = (kWave / LPH) >> p.slot_heads_log2, groups = per_wave * kWavesPerBlock;
  const int group = (slot >> p.slot_heads_log2) + per_wave * (threadIdx.x >> 6);
  t.head = ((int)blockIdx.y << p.slot_heads_log2) + hs;
  t.d0 = piece * N;
  t.n = t.head < heads ? p.dim - t.d0 : 0;
  t.write = true;
  float a[N] = {}, b[N] = {}, rest = 0.0f;
  if (t.n > 0)
    for (int64_t c = blockIdx.x + group; c <= last; c += groups) {
      const float *part = p.part + (c * 2 + (c == blockIdx.x)) * p.part_floats + (int64_t)t.head * (2 * LPH * N + 1);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        a[i] += part[t.d0 + i];
        b[i] += part[LPH * N + t.d0 + i];
      }
      if (!COLUMNS) rest += part[2 * LPH * N];
    }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    sh[threadIdx.x][i] = a[i];
    sh[threadIdx.x][N + i] = b[i];
  }
  sh[threadIdx.x][2 * N] = rest;
  float g[N], m, r, d0;
  if (!COLUMNS && group == 0) load_row<T, LPH, WIDE>(p, t, g, m, r, d0);
  __syncthreads();
  if (group != 0 || t.n <= 0) return;
  for (int o = 1; o < groups; ++o) {
    const float *other = sh[(o / per_wave) * kWave + (((o % per_wave) << p.slot_heads_log2) + hs) * LPH + piece];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a[i] += other[i];
      b[i] += other[N + i];
    }
    rest += other[2 * N];
  }
  if constexpr (COLUMNS) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] *= p.scale;
    store_piece<T, WIDE>((T *)p.o0 + t.row * p.o0_row + t.head * p.o0_head + t.d0, t.n, a);
    store_piece<T, WIDE>((T *)p.o1 + t.row * p.o1_row + t.head * p.o1_head + t.d0, t.n, b);
  } else {
    finish_rows<T, WIDE>(p, t, m, r, d0, rest, a, b);
  }
}

// ------------------------------------------------------------------ host side
enum { kForward = 0, kBackwardRows = 1, kBackwardColumns = 2 };

static int log2_ceil(int64_t x) {
  int l = 0;
  while (((int64_t)1 << l) < x) ++l;
  return l;
}

static int lanes_per_head(int dtype, int dim) {
  return 1 << log2_ceil(ceil_div(dim, dtype == GCNX_F32 ? 4 : 8));
}

static int64_t part_floats(int pass, int dtype, int heads, int kv_heads, int dim) {
  const int64_t wide = (int64_t)lanes_per_head(dtype, dim) * (dtype == GCNX_F32 ? 4 : 8);
  return pass == kForward ? heads * (wide + 2) : (pass == kBackwardRows ? heads : kv_heads) * (2 * wide + 1);
}

static bool rows_are_cut(int64_t nnz, int64_t max_row_nnz) {
  return nnz > kSegment && (max_row_nnz <= 0 || max_row_nnz > kSegment);
}

template <typename T, int LPH, bool WIDE>
static void launch_pass(int pass, AttnArgs p, hipStream_t stream) {
  const int heads = pass == kBackwardColumns ? p.kv_heads : p.heads;
  const int slots_log2 = log2_ceil(kWave / LPH);
  const int heads_log2 = log2_ceil(heads);
  p.slot_heads_log2 = heads_log2 < slots_log2 ? heads_log2 : slots_log2;
  const int spare = slots_log2 - p.slot_heads_log2;
  // edges side by side: about kUnroll per lane at the average row; what is left
  // takes further rows
  const int64_t items = ceil_div(p.nnz * (pass == kBackwardColumns ? p.group : 1), p.n_rows);
  int e = log2_ceil(ceil_div(items, kUnroll));
  p.edge_log2 = e < spare ? e : spare;
  p.row_log2 = spare - p.edge_log2;
  const int64_t tasks = p.n_pieces + ceil_div(p.n_rows, (int64_t)1 << p.row_log2);
  const dim3 grid((unsigned)ceil_div(tasks, kWavesPerBlock), (unsigned)ceil_div(heads, (int64_t)1 << p.slot_heads_log2));
  const dim3 joins((unsigned)(p.n_pieces / 2), grid.y);
  if (pass == kForward) {
    hipLaunchKernelGGL((attention_forward_kernel<T, LPH, WIDE>), grid, dim3(kBlock), 0, stream, p);
    if (p.n_pieces) hipLaunchKernelGGL((attention_forward_join_kernel<T, LPH, WIDE>), joins, dim3(kBlock), 0, stream, p);
  } else if (pass == kBackwardRows) {
    hipLaunchKernelGGL((attention_backward_rows_kernel<T, LPH, WIDE>), grid, dim3(kBlock), 0, stream, p);
    if (p.n_pieces) hipLaunchKernelGGL((attention_backward_join_kernel<T, LPH, WIDE, false>), joins, dim3(kBlock), 0, stream, p);
  } else {
    hipLaunchKernelGGL((attention_backward_columns_kernel<T, LPH, WIDE>), grid, dim3(kBlock), 0, stream, p);
    if (p.n_pieces) hipLaunchKernelGGL((attention_backward_join_kernel<T, LPH, WIDE, true>), joins, dim3(kBlock), 0, stream, p);
  }
}

template <typename T, bool WIDE>
static void launch_lanes(int pass, int lph, const AttnArgs &p, hipStream_t stream) {
  switch (lph) {
    case 1: return launch_pass<T, 1, WIDE>(pass, p, stream);
    case 2: return launch_pass<T, 2, WIDE>(pass, p, stream);
    case 4: return launch_pass<T, 4, WIDE>(pass, p, stream);
    case 8: return launch_pass<T, 8, WIDE>(pass, p, stream);
    case 16: return launch_pass<T, 16, WIDE>(pass, p, stream);
    case 32: return launch_pass<T, 32, WIDE>(pass, p, stream);
    default:
      if constexpr (Piece<T>::N == 4) return launch_pass<T, 64, WIDE>(pass, p, stream);
  }
}

template <typename T>
static void launch_type(int pass, bool wide, int lph, const AttnArgs &p, hipStream_t stream) {
  if (wide) launch_lanes<T, true>(pass, lph, p, stream);
  else launch_lanes<T, false>(pass, lph, p, stream);
}

static int launch(int pass, int dtype, bool wide, AttnArgs p, hipStream_t stream) {
  if (p.n_rows == 0) return GCNX_OK;
  const int lph = lanes_per_head(dtype, p.dim);
  if (dtype == GCNX_F32) launch_type<float>(pass, wide, lph, p, stream);
  else if (dtype == GCNX_BF16) launch_type<__bf16>(pass, wide, lph, p, stream);
  else launch_type<_Float16>(pass, wide, lph, p, stream);
  GCNX_CHECK_LAUNCH();
  return GCNX_OK;
}

static int check(const gcnx_attention *p) {
  GCNX_REQUIRE(p && p->a, GCNX_ERR_INVALID_ARG, "attention: null argument");
  GCNX_REQUIRE(p->dtype == GCNX_F32 || p->dtype == GCNX_BF16 || p->dtype == GCNX_F16, GCNX_ERR_UNSUPPORTED,
               "attention: dtype %d", p->dtype);
  GCNX_REQUIRE(p->head_dim >= 1 && p->head_dim <= 256, GCNX_ERR_UNSUPPORTED, "attention: head_dim %d outside 1..256",
               p->head_dim);
  GCNX_REQUIRE(p->n_kv_heads >= 1 && p->n_heads >= 1 && p->n_heads % p->n_kv_heads == 0 && p->n_heads <= 65535,
               GCNX_ERR_INVALID_ARG, "attention: %d query heads over %d key heads", p->n_heads, p->n_kv_heads);
  GCNX_REQUIRE(p->a->n_rows >= 0 && p->a->n_cols >= 0 && p->a->nnz >= 0 && p->a->n_rows < 2147483647 &&
                   p->a->nnz / kSegment < 1000000000, GCNX_ERR_INVALID_ARG, "attention: bad matrix size");
  GCNX_REQUIRE((p->a->n_rows == 0 || p->a->row_ptr) && (p->a->nnz == 0 || p->a->col_idx), GCNX_ERR_INVALID_ARG,
               "attention: null matrix array");
  GCNX_REQUIRE(p->a->nnz == 0 || (p->a->n_rows > 0 && p->a->n_cols > 0), GCNX_ERR_INVALID_ARG, "attention: nonzeros in an empty matrix");
  GCNX_REQUIRE(!p->use_values || p->a->nnz == 0 || p->a->val, GCNX_ERR_INVALID_ARG, "attention: values asked for, none given");
  GCNX_REQUIRE((p->a->n_rows == 0 || p->q) && (p->a->n_cols == 0 || (p->k && p->v)), GCNX_ERR_INVALID_ARG,
               "attention: null operand");
  GCNX_REQUIRE(p->q_row >= 0 && p->q_head >= 0 && p->k_row >= 0 && p->k_head >= 0 && p->v_row >= 0 && p->v_head >= 0,
               GCNX_ERR_INVALID_ARG, "attention: negative stride");
  return GCNX_OK;
}

// 16-byte loads of every piece: base and strides multiples of 16 bytes.
static bool piece_aligned(const gcnx_attention *p, const void *base, int64_t row, int64_t head) {
  const int64_t n = p->dtype == GCNX_F32 ? 4 : 8;
  return p->head_dim % n == 0 && row % n == 0 && head % n == 0 && ((uintptr_t)base & 15) == 0;
}

static AttnArgs common_args(const gcnx_attention *p) {
  AttnArgs g = {};
  g.q = p->q; g.q_row = p->q_row; g.q_head = p->q_head;
  g.k = p->k; g.k_row = p->k_row; g.k_head = p->k_head;
  g.v = p->v; g.v_row = p->v_row; g.v_head = p->v_head;
  g.heads = p->n_heads;
  g.kv_heads = p->n_kv_heads;
  g.group = p->n_heads / p->n_kv_heads;
  g.dim = p->head_dim;
  g.scale = p->scale;
  return g;
}

static void set_pattern(AttnArgs &g, const gcnx_attention *p, const gcnx_csr *a, const int32_t *chunk_row,
                        const int64_t *mask_index, int64_t max_row_nnz, int pass, float *part) {
  g.row_ptr = a->row_ptr;
  g.col_idx = a->col_idx;
  g.val = p->use_values ? a->val : nullptr;
  g.mask = p->edge_mask;
  g.mask_index = mask_index;
  g.chunk_row = chunk_row;
  g.n_rows = a->n_rows;
  g.nnz = a->nnz;
  g.part = part;
  g.part_floats = part_floats(pass, p->dtype, p->n_heads, p->n_kv_heads, p->head_dim);
  g.n_pieces = rows_are_cut(a->nnz, max_row_nnz) ? 2 * ceil_div(a->nnz, kSegment) : 0;
}

static size_t part_bytes(const gcnx_attention *p, int64_t max_row_nnz, int pass) {
  if (!rows_are_cut(p->a->nnz, max_row_nnz)) return 0;
  return align_up((size_t)(2 * ceil_div(p->a->nnz, kSegment)) *
                      part_floats(pass, p->dtype, p->n_heads, p->n_kv_heads, p->head_dim) * sizeof(float), 256);
}

static size_t stats4_bytes(const gcnx_attention *p) {
  return align_up((size_t)p->a->n_rows * p->n_heads * 16, 256);
}

}  // namespace gcnx

using namespace gcnx;

extern "C" size_t gcnx_attention_workspace_bytes(const gcnx_attention *p) {
  if (check(p) != GCNX_OK) return 0;
  return part_bytes(p, p->max_row_nnz, kForward);
}

extern "C" int gcnx_attention_forward(const gcnx_attention *p, const int32_t *chunk_row, void *out, int64_t out_row,
                                      int64_t out_head, float *stats, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check(p)) return rc;
  if (p->a->n_rows == 0) return GCNX_OK;
  GCNX_REQUIRE(out && out_row >= 0 && out_head >= 0, GCNX_ERR_INVALID_ARG, "attention: bad output");
  const size_t need = part_bytes(p, p->max_row_nnz, kForward);
  GCNX_REQUIRE(need == 0 || (chunk_row && ws && ws_bytes >= need), GCNX_ERR_WORKSPACE,
               "attention: workspace of %zu bytes (and the chunk table) needed, %zu given", need, ws_bytes);
  AttnArgs g = common_args(p);
  set_pattern(g, p, p->a, chunk_row, p->mask_index, p->max_row_nnz, kForward, (float *)ws);
  g.o0 = out; g.o0_row = out_row; g.o0_head = out_head;
  g.stats = stats;
  const bool wide = piece_aligned(p, p->q, p->q_row, p->q_head) && piece_aligned(p, p->k, p->k_row, p->k_head) &&
                    piece_aligned(p, p->v, p->v_row, p->v_head) && piece_aligned(p, out, out_row, out_head);
  return launch(kForward, p->dtype, wide, g, as_stream(stream));
}

extern "C" size_t gcnx_attention_backward_workspace_bytes(const gcnx_attention *p, int64_t t_max_row_nnz) {
  if (check(p) != GCNX_OK) return 0;
  const size_t rows = part_bytes(p, p->max_row_nnz, kBackwardRows), cols = part_bytes(p, t_max_row_nnz, kBackwardColumns);
  return stats4_bytes(p) + (rows > cols ? rows : cols);
}

extern "C" int gcnx_attention_backward(const gcnx_attention *p, const int32_t *chunk_row, const gcnx_csr *at,
                                       const int32_t *t_chunk_row, const int64_t *t_mask_index, int64_t t_max_row_nnz,
                                       const void *out, int64_t out_row, int64_t out_head, const float *stats,
                                       const void *dout, int64_t dout_row, int64_t dout_head, void *dq, void *dk,
                                       void *dv, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check(p)) return rc;
  GCNX_REQUIRE(at && at->n_rows == p->a->n_cols && at->n_cols == p->a->n_rows && at->nnz == p->a->nnz,
               GCNX_ERR_INVALID_ARG, "attention: the transpose does not belong to the matrix");
  GCNX_REQUIRE((at->n_rows == 0 || at->row_ptr) && (at->nnz == 0 || (at->col_idx && (!p->use_values || at->val))),
               GCNX_ERR_INVALID_ARG, "attention: null array in the transpose");
  GCNX_REQUIRE(!p->edge_mask || at->nnz == 0 || t_mask_index, GCNX_ERR_INVALID_ARG,
               "attention: the mask needs its index in the transpose");
  GCNX_REQUIRE(p->a->n_rows == 0 || (out && dout && stats && out_row >= 0 && out_head >= 0 && dout_row >= 0 && dout_head >= 0),
               GCNX_ERR_INVALID_ARG, "attention: bad output or gradient of it");
  GCNX_REQUIRE((dk == nullptr) == (dv == nullptr) && (dq || dk || (p->a->n_rows == 0 && p->a->n_cols == 0)),
               GCNX_ERR_INVALID_ARG, "attention: dq, or dk and dv, or all three");
  const size_t need = gcnx_attention_backward_workspace_bytes(p, t_max_row_nnz);
  GCNX_REQUIRE(need == 0 || (ws && ws_bytes >= need), GCNX_ERR_WORKSPACE,
               "attention: workspace of %zu bytes needed, %zu given", need, ws_bytes);
  GCNX_REQUIRE((!rows_are_cut(p->a->nnz, p->max_row_nnz) || chunk_row) &&
                   (!rows_are_cut(p->a->nnz, t_max_row_nnz) || t_chunk_row), GCNX_ERR_INVALID_ARG,
               "attention: chunk table needed");
  const int64_t hd = (int64_t)p->n_heads * p->head_dim, kd = (int64_t)p->n_kv_heads * p->head_dim;
  const bool reads = piece_aligned(p, p->q, p->q_row, p->q_head) && piece_aligned(p, p->k, p->k_row, p->k_head) &&
                     piece_aligned(p, p->v, p->v_row, p->v_head) && piece_aligned(p, dout, dout_row, dout_head);
  AttnArgs g = common_args(p);
  g.out = out; g.out_row = out_row; g.out_head = out_head;
  g.dout = dout; g.dout_row = dout_row; g.dout_head = dout_head;
  g.stats = const_cast<float *>(stats);
  g.stats4 = (f32x4 *)ws;
  float *part = (float *)((char *)ws + stats4_bytes(p));
  set_pattern(g, p, p->a, chunk_row, p->mask_index, p->max_row_nnz, kBackwardRows, part);
  g.o0 = dq; g.o0_row = hd; g.o0_head = p->head_dim;
  if (int rc = launch(kBackwardRows, p->dtype, reads && piece_aligned(p, out, out_row, out_head) &&
                                                   piece_aligned(p, dq, hd, p->head_dim), g, as_stream(stream)))
    return rc;
  if (!dk) return GCNX_OK;
  set_pattern(g, p, at, t_chunk_row, t_mask_index, t_max_row_nnz, kBackwardColumns, part);
  g.o0 = dk; g.o0_row = kd; g.o0_head = p->head_dim;
  g.o1 = dv; g.o1_row = kd; g.o1_head = p->head_dim;
  return launch(kBackwardColumns, p->dtype, reads && piece_aligned(p, dk, kd, p->head_dim) && piece_aligned(p, dv, kd, p->head_dim),
                g, as_stream(stream));
}
