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
// What bounds it: k and v of every edge are read through the caches, and where every
// query head has its own keys 4 (7 or 10 backward) flops an element gathered leave the
// matrix units nothing to do.  (Heads that share keys gather less and compute the same:
// there the vector ALU bounds the forward and the row pass, 70 to 75 % busy at 8 on 2;
// their scores are products of a kind that the matrix units could take.)  2^19 nodes, 8.9 M
// edges, 8 heads of 32, bf16: forward 1.03 ms, row pass 1.15, column pass 1.25 for 9.1,
// 9.1 and 10.3 GB gathered; a quarter of it hits L2, the rest comes at 6.4 to 6.8 TB/s,
// what the fabric behind the L2s gives.  Operands within the caches: 2^16 nodes, forward
// 0.10 ms, 11 TB/s.  Hence the layout: a head's vector lies in 16-byte pieces across
// neighbouring lanes (a key row is one coalesced read), the lanes of a wavefront are
// edges x heads, an edge is read once for its score and its value, and the next edge's
// index and operands are under way while the present one is summed.
//
// m and r are kept instead of the one number m - log r: at logits of 10^4, or a row
// whose every value is the type's lowest, fp32 has no digits left for log r.
#include "gcnx_common.h"
#include "gcnx_piece.h"

namespace gcnx {

// <a, b> + c over a piece.  16 bits: two exact products and their sum an instruction.
template <typename T>
__device__ __forceinline__ float dot_piece(const typename Piece<T>::raw &a, const typename Piece<T>::raw &b) {
  float d = 0.0f;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) d = fmaf(a[i], b[i], d);
  } else {
    typedef T pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const pair x = {a[2 * i], a[2 * i + 1]}, y = {b[2 * i], b[2 * i + 1]};
      if constexpr (sizeof(T) == 2 && __is_same(T, _Float16)) d = __builtin_amdgcn_fdot2(x, y, d, false);
      else d = __builtin_amdgcn_fdot2_f32_bf16(x, y, d, false);
    }
  }
  return d;
}

// A piece without the elements that another lane counts, or that there are none of.
template <typename T, int LPH>
__device__ __forceinline__ typename Piece<T>::raw counted(typename Piece<T>::raw x, int skip, int dim) {
#pragma unroll
  for (int i = 0; i < Piece<T>::N; ++i)
    if (LPH ? i < skip : i >= dim) x[i] = (T)0.0f;
  return x;
}

// The sums over a head of own * x and of own2 * x2.  RAGGED: a head that is no multiple
// of a piece.  The lane's own operand is zero where it does not count, which leaves
// the other side's element out unless that is not finite: 0 * inf.  A NaN of that
// origin cannot be told from another by the sum, so the products of a wavefront that
// meets one are formed again with zeros on both sides.  (Zeros on both sides for
// every edge: backward of 4.2 M edges at 8 x 20 bf16 1140 us against 1040, at 4 x 5
// 1303 against 1066.)
template <typename T, int LPH, bool RAGGED>
__device__ __forceinline__ float head_dot(const typename Piece<T>::raw &own, const typename Piece<T>::raw &x, int skip, int dim) {
  float s = group_sum<LPH>(dot_piece<T>(own, x));
  if constexpr (RAGGED)
    if (__any(s != s)) s = group_sum<LPH>(dot_piece<T>(own, counted<T, LPH>(x, skip, dim)));
  return s;
}
template <typename T, int LPH, bool RAGGED>
__device__ __forceinline__ f32x2 head_dots(const typename Piece<T>::raw &own, const typename Piece<T>::raw &x, const typename Piece<T>::raw &own2,
                                           const typename Piece<T>::raw &x2, int skip, int dim) {
  float s = group_sum<LPH>(dot_piece<T>(own, x)), d = group_sum<LPH>(dot_piece<T>(own2, x2));
  if constexpr (RAGGED)
    if (__any(s != s || d != d)) {
      s = group_sum<LPH>(dot_piece<T>(own, counted<T, LPH>(x, skip, dim)));
      d = group_sum<LPH>(dot_piece<T>(own2, counted<T, LPH>(x2, skip, dim)));
    }
  return f32x2{s, d};
}

__device__ __forceinline__ bool is_lowest(float x) { return x == -__builtin_inff(); }

// Edges in flight per lane: more cost registers, so wavefronts, and idle slots at the
// ends of rows.  1 / 2 / 4, us at 2^19 nodes: forward 1082 / 1057 / 1075, row pass
// 1176 / 1257 / 1406, column pass 1317 / 1394 / 1645.
constexpr int kForwardEdges = 2;
constexpr int kBackwardEdges = 1;

// Wavefronts a SIMD that the registers have to leave room for: 8 (64 registers) where
// nothing is spilled for it.  (Column pass at 2^19 nodes: 1284 us against 1525 with
// the 5 that the compiler chooses.)
template <int LPH, bool SHIFTS>
constexpr int kWaves = SHIFTS && LPH == 0 ? 5 : SHIFTS || LPH == 0 || LPH >= 32 ? 6 : 8;

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
  uint32_t q_bytes, q_head_bytes, k_bytes, v_bytes, dout_bytes, dout_head_bytes;   // the same strides where rows are gathered
  int32_t heads, kv_heads, group, dim;
  float scale;
  // results
  void *o0, *o1;
  int64_t o0_row, o0_head, o1_row, o1_head;
  float *stats;                 // forward: 2 per row and head; backward row pass reads them
  f32x4 *stats4;                // backward: m, r, delta per row and head
  // work split
  float *part;                  // partial results of cut rows
  int64_t part_floats;          // per piece; 0: no pieces
  int64_t n_pieces;             // tasks of cut rows, before those of the others
  bool whole;                   // a cut row is one workgroup's (4 tasks a chunk), else pieces (2 tasks a chunk)
  int32_t segment;              // rows longer than this are cut at its multiples
  int32_t heads_log2;           // heads side by side in a wavefront (a tile)
  int32_t edge_log2, row_log2;  // edges of a row, rows side by side in a wavefront
  int32_t tiles, tiles_log2;    // tiles_log2 < 0: no power of two up to 8
};

// What one group of lanes works on.
struct Task {
  int64_t row, beg;
  uint32_t count;               // edges from beg on
  int64_t piece;                // >= 0: a piece of a cut row
  bool whole;                   // the workgroup's wavefronts share the row
  bool live;                    // the lane has a head and a row to write
  int32_t edge, edges;          // this lane's first edge, and the edges read side by side
  int32_t side;                 // of them in this wavefront
  bool first;                   // the lane that holds the wavefront's sums
  int32_t head, d0, skip;       // head, first element of the lane's piece, elements counted by another lane
};

// Tile of heads and place in its list of tasks.  Workgroups go to the 8 dies in
// turn; tiles are dealt so that a die sees one tile only (or as few as there are):
// its L2 then holds the operand rows of that tile's heads alone.
__device__ __forceinline__ int64_t tile_of(const AttnArgs &p, int &tile) {
  const uint32_t id = blockIdx.x;
  if (p.tiles_log2 >= 0) {
    const uint32_t die = id & 7;
    tile = die & (p.tiles - 1);
    return ((int64_t)(id >> 3) << (3 - p.tiles_log2)) + (die >> p.tiles_log2);
  }
  tile = id % p.tiles;
  return id / p.tiles;
}

template <typename T, int LPH>
__device__ __forceinline__ void place_lane(const AttnArgs &p, int heads, int tile, Task &t, int &slot) {
  constexpr int L = LPH ? LPH : 1, N = Piece<T>::N;
  const int lane = threadIdx.x & (kWave - 1), piece = lane % L;
  slot = lane / L;
  t.head = (tile << p.heads_log2) + (slot & ((1 << p.heads_log2) - 1));
  t.d0 = piece * N;
  t.skip = 0;
  t.live = t.head < heads && t.d0 < p.dim;
  if (LPH && t.d0 + N > p.dim) {
    t.skip = t.d0 < p.dim ? t.d0 + N - p.dim : N;
    t.d0 = p.dim - N;
  }
  slot >>= p.heads_log2;
}

template <typename T, int LPH>
__device__ __forceinline__ bool find_task(const AttnArgs &p, int heads, Task &t) {
  constexpr int L = LPH ? LPH : 1;
  int tile, slot;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);     // tasks are in scalar registers
  const int64_t task = tile_of(p, tile) * kWavesPerBlock + wave;
  place_lane<T, LPH>(p, heads, tile, t, slot);
  int64_t end;
  t.piece = -1;
  t.whole = false;
  t.first = slot == 0;
  if (task < p.n_pieces) {
    t.side = (kWave / L) >> p.heads_log2;
    t.whole = p.whole;
    t.edge = p.whole ? slot + wave * t.side : slot;
    t.edges = p.whole ? t.side * kWavesPerBlock : t.side;
    const int64_t first = (p.whole ? task >> 2 : task >> 1) * p.segment, next = first + p.segment;
    if (p.whole || (task & 1)) {        // the cut row that begins in this chunk
      if (next >= p.nnz) return false;
      t.row = p.chunk_row[next / kChunkUnit];
      t.beg = p.row_ptr[t.row];
      end = p.row_ptr[t.row + 1];
      if (t.beg < first || t.beg >= next || end - t.beg <= p.segment) return false;
      if (!p.whole) end = next;
    } else {                            // the cut row that goes on into this chunk
      t.row = p.chunk_row[first / kChunkUnit];
      t.beg = p.row_ptr[t.row];
      end = p.row_ptr[t.row + 1];
      if (t.beg >= first || end - t.beg <= p.segment) return false;
      t.beg = first;
      end = end < next ? end : next;
    }
    if (!p.whole) t.piece = task;
  } else {
    t.edge = slot & ((1 << p.edge_log2) - 1);
    t.side = t.edges = 1 << p.edge_log2;
    t.first = t.edge == 0;
    t.row = ((task - p.n_pieces) << p.row_log2) + (slot >> p.edge_log2);
    const bool there = t.row < p.n_rows;
    if (!there) t.row = p.n_rows - 1;
    t.beg = p.row_ptr[t.row];
    end = p.row_ptr[t.row + 1];
    if (!there || (p.n_pieces && end - t.beg > p.segment)) {
      t.live = false;
      end = t.beg;            // for every lane of the group: its sums need them all
    }
  }
  t.count = (uint32_t)(end - t.beg);
  return true;
}

// An edge, read a turn before it is used: its column, its logit shift, whether it
// takes part.  An edge whose shift is -inf is out of the softmax like a masked one:
// its operands are not read, so infinities and NaN in masked places stay where they
// are.  SHIFTS: there are values or a mask; the mask's index is then read two turns
// ahead, its byte one.  What is read is not looked at before its turn, so that
// nothing waits for it.
template <bool SHIFTS>
struct Edge {
  int32_t col;
  float shift;
  uint32_t keep;
  bool there;
  int64_t index;
  __device__ __forceinline__ void start(const AttnArgs &p, const Task &t, uint32_t x) {
    there = x < t.count;
    const int64_t e = t.beg + (there ? x : 0);       // t.count > 0: edge 0 is there
    col = p.col_idx[e];
    shift = 0.0f;
    keep = 1;
    if constexpr (SHIFTS) {
      if (p.val) shift = p.val[e];
      index = e;
      if (p.mask_index) index = p.mask_index[e];
    }
  }
  __device__ __forceinline__ void check(const AttnArgs &p) {
    if constexpr (SHIFTS)
      if (p.mask) keep = p.mask[index];
  }
  __device__ __forceinline__ bool on() const { return there && (!SHIFTS || (keep != 0 && !is_lowest(shift))); }
};

// U edges a turn; place(u) is the place in the row of the u-th edge to read.
template <bool SHIFTS, int U>
struct Edges {
  Edge<SHIFTS> next[U], later[U];
  __device__ __forceinline__ bool more() const { return next[0].there; }
  template <typename Place>
  __device__ __forceinline__ void begin(const AttnArgs &p, const Task &t, Place place) {
#pragma unroll
    for (int u = 0; u < U; ++u) next[u].start(p, t, place(u));
    if constexpr (SHIFTS) {
#pragma unroll
      for (int u = 0; u < U; ++u) later[u].start(p, t, place(U + u));
#pragma unroll
      for (int u = 0; u < U; ++u) next[u].check(p);
    }
  }
  // place(u): of the edge that comes `ahead` turns after this one
  static constexpr int ahead = SHIFTS ? 2 : 1;
  template <typename Place>
  __device__ __forceinline__ void advance(const AttnArgs &p, const Task &t, Place place) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (SHIFTS) {
        next[u] = later[u];
        later[u].start(p, t, place(u));
      } else {
        next[u].start(p, t, place(u));
      }
    }
    if constexpr (SHIFTS) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u].check(p);
    }
  }
};

// The lane's own operand; elements that another lane counts are zero.
template <typename T, int LPH>
__device__ __forceinline__ typename Piece<T>::raw load_own(const AttnArgs &p, const Task &t, const void *base, int64_t row, int64_t head) {
  const Address at = (Address)((const T *)base + t.row * row + t.head * head + t.d0);
  typename Piece<T>::raw x = load_piece<T, LPH == 0>(at_or_zeros(at, t.live), p.dim);
#pragma unroll
  for (int i = 0; i < Piece<T>::N; ++i)
    if (LPH ? i < t.skip : i >= p.dim) x[i] = (T)0.0f;
  return x;
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

template <typename T, int LPH, int N>
__device__ __forceinline__ void finish_forward(const AttnArgs &p, const Task &t, float m, float l, const float (&acc)[N]) {
  const float r = l == 0.0f ? 0.0f : 1.0f / l;      // nothing takes part: zeros
  float o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = acc[i] * r;
  store_piece<T, LPH == 0>((T *)p.o0 + t.row * p.o0_row + t.head * p.o0_head + t.d0, p.dim, o);
  if (p.stats && t.d0 == 0) {
    float *st = p.stats + (t.row * p.heads + t.head) * 2;
    st[0] = is_lowest(m) ? 0.0f : m;
    st[1] = r;
  }
}

// Elements of a partial vector of one head in the workspace: the vector (two in the
// backward passes), then four numbers, of which two (one) are used.
template <typename T, int LPH>
constexpr int kPartWide = (LPH ? LPH : 1) * Piece<T>::N;

template <typename T, int LPH, bool SHIFTS, bool RAGGED>
__global__ __launch_bounds__(kBlock, (kWaves<LPH, SHIFTS>)) void attention_forward_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N;
  typedef typename Piece<T>::raw raw;
  __shared__ float sh[N + 2][kWave];
  Task t;
  if (!find_task<T, LPH>(p, p.heads, t)) return;
  const int kv = t.head / p.group;
  const raw q = load_own<T, LPH>(p, t, p.q, p.q_row, p.q_head);
  float acc[N] = {}, m = -__builtin_inff(), l = 0.0f;
  const Address kb = (Address)((const T *)p.k + kv * p.k_head + t.d0), vb = (Address)((const T *)p.v + kv * p.v_head + t.d0);
  if (t.count) {
    Edges<SHIFTS, kForwardEdges> edges;
    edges.begin(p, t, [&](int u) { return t.edge + u * t.edges; });
    for (uint32_t x = t.edge; edges.more(); x += kForwardEdges * t.edges) {
      raw k[kForwardEdges], v[kForwardEdges];
      float s[kForwardEdges];
      bool on[kForwardEdges];
#pragma unroll
      for (int u = 0; u < kForwardEdges; ++u) {
        on[u] = edges.next[u].on();
        s[u] = edges.next[u].shift;
        k[u] = load_piece<T, LPH == 0>(at_or_zeros(row_at(kb, edges.next[u].col, p.k_bytes), on[u] && t.live), p.dim);
        v[u] = load_piece<T, LPH == 0>(at_or_zeros(row_at(vb, edges.next[u].col, p.v_bytes), on[u] && t.live), p.dim);
      }
      edges.advance(p, t, [&](int u) { return x + (edges.ahead * kForwardEdges + u) * t.edges; });
      read_ahead_fence();
      float top = m;
#pragma unroll
      for (int u = 0; u < kForwardEdges; ++u) {
        const float d = head_dot<T, LPH, RAGGED>(q, k[u], t.skip, p.dim);
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
      for (int u = 0; u < kForwardEdges; ++u) {
        const float w = exp_of(s[u] - safe);
        l += w;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(w, (float)v[u][i], acc[i]);
      }
    }
  }
  for (int at = 1; at < t.side; at <<= 1) {
    const int off = ((LPH ? LPH : 1) * at) << p.heads_log2;
    float m2 = __shfl_xor(m, off, kWave), l2 = __shfl_xor(l, off, kWave), acc2[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc2[i] = __shfl_xor(acc[i], off, kWave);
    join<N>(m, l, acc, m2, l2, acc2);
  }
  if (t.whole) {
    // All wavefronts of the workgroup are here: theirs are joined to the first one's,
    // one after the other through one small buffer (LDS is held until the last
    // wavefront of a workgroup ends, so much of it would keep others out).
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & (kWave - 1);
    for (int w = 1; w < kWavesPerBlock; ++w) {
      if (wave == w) {
        sh[0][lane] = m;
        sh[1][lane] = l;
#pragma unroll
        for (int i = 0; i < N; ++i) sh[2 + i][lane] = acc[i];
      }
      __syncthreads();
      if (wave == 0) {
        float a2[N];
#pragma unroll
        for (int i = 0; i < N; ++i) a2[i] = sh[2 + i][lane];
        join<N>(m, l, acc, sh[0][lane], sh[1][lane], a2);
      }
      __syncthreads();
    }
    if (wave != 0) return;
  }
  if (!t.first || !t.live) return;
  if (t.piece >= 0) {
    float *part = p.part + t.piece * p.part_floats + (int64_t)t.head * (kPartWide<T, LPH> + 4);
    store_floats<N>(part + t.d0, acc);
    if (t.d0 == 0) {
      part[kPartWide<T, LPH>] = m;
      part[kPartWide<T, LPH> + 1] = l;
    }
    return;
  }
  finish_forward<T, LPH, N>(p, t, m, l, acc);
}

// Joining the pieces of cut rows: those that begin in one of kJoinChunks chunks, a
// tile of heads of them, by a workgroup.  A row's pieces are slot 1 of the chunk that
// it begins in and slot 0 of the chunks after it.  Rows of up to kJoinWave pieces are
// dealt to the wavefronts, longer ones are the whole workgroup's.  The pieces of a row
// are dealt to groups of lanes, kJoinAhead read at a time; each group joins its own in
// order, then groups are joined by exchanges in the wavefront and (for the workgroup's
// rows) through LDS: a fixed tree.
// Latency bounds it.  us of the backward pass's join, every row the workgroup's and 4
// chunks -> this: 8.5 M edges of 2^19 rows 40 -> 25 (columns 29 -> 21), 0.9 M edges of
// heads 8 on 2 x 64 31 -> 28 (17 -> 10), 2^20 edges of 3 rows 23 -> 17.  16 chunks: the
// same within 2 us; kJoinWave 32: the same.
constexpr int kJoinChunks = 8;
constexpr int kJoinWave = 16;
constexpr int kJoinAhead = 4;

struct JoinTask {
  int64_t first, last;          // chunks of the row
  __device__ __forceinline__ const float *part(const AttnArgs &p, int64_t c) const {
    return p.part + ((c <= last ? c : last) * 2 + (c == first)) * p.part_floats;
  }
};

// Which of the workgroup's chunks have a cut row begin in them, a lane a chunk; row
// and last chunk of the lane's.
__device__ __forceinline__ uint64_t find_joins(const AttnArgs &p, int64_t &row, int64_t &last, uint64_t &small) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t first = ((int64_t)blockIdx.x * kJoinChunks + lane) * p.segment, next = first + p.segment;
  bool found = false;
  row = last = 0;
  if (lane < kJoinChunks && next < p.nnz) {
    row = p.chunk_row[next / kChunkUnit];
    const int64_t beg = p.row_ptr[row], end = p.row_ptr[row + 1];
    last = (end - 1) / p.segment;
    found = beg >= first && beg < next && end - beg > p.segment;
  }
  small = __ballot(found && last - (next / p.segment - 1) < kJoinWave);
  return __ballot(found);
}

template <typename T, int LPH>
__global__ __launch_bounds__(kBlock) void attention_forward_join_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N, L = LPH ? LPH : 1;
  const int span = L << p.heads_log2;        // lanes of a group
  __shared__ float sh[kWavesPerBlock][kWave][N + 2];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  Task t;
  JoinTask j;
  int slot;
  place_lane<T, LPH>(p, p.heads, blockIdx.y, t, slot);
  const int head = t.live ? t.head : 0;      // lanes behind the last head read along
  int64_t rows, lasts;
  uint64_t small;
  const uint64_t found = find_joins(p, rows, lasts, small);
  const auto join_row = [&](int chunk, bool block) {
    const int groups = (block ? kBlock : kWave) / span, group = (block ? threadIdx.x : lane) / span;
    t.row = __shfl(rows, chunk, kWave);
    j.first = (int64_t)blockIdx.x * kJoinChunks + chunk;
    j.last = __shfl(lasts, chunk, kWave);
    float m = -__builtin_inff(), l = 0.0f, acc[N] = {};
    for (int64_t c = j.first + group; c <= j.last; c += kJoinAhead * groups) {
      float m2[kJoinAhead], l2[kJoinAhead], a2[kJoinAhead][N];
#pragma unroll
      for (int u = 0; u < kJoinAhead; ++u) {
        const float *part = j.part(p, c + u * groups) + (int64_t)head * (kPartWide<T, LPH> + 4);
        m2[u] = part[kPartWide<T, LPH>];
        l2[u] = part[kPartWide<T, LPH> + 1];
        load_floats<N>(part + t.d0, a2[u]);
      }
#pragma unroll
      for (int u = 0; u < kJoinAhead; ++u)
        if (c + u * groups <= j.last) join<N>(m, l, acc, m2[u], l2[u], a2[u]);
    }
    for (int off = span; off < kWave; off <<= 1) {
      float m2 = __shfl_xor(m, off, kWave), l2 = __shfl_xor(l, off, kWave), a2[N];
#pragma unroll
      for (int i = 0; i < N; ++i) a2[i] = __shfl_xor(acc[i], off, kWave);
      join<N>(m, l, acc, m2, l2, a2);
    }
    if (block) {
      __syncthreads();
      if (lane < span) {
        sh[wave][lane][0] = m;
        sh[wave][lane][1] = l;
#pragma unroll
        for (int i = 0; i < N; ++i) sh[wave][lane][2 + i] = acc[i];
      }
      __syncthreads();
      if (wave != 0) return;
      if (lane < span)
#pragma unroll
        for (int w = 1; w < kWavesPerBlock; ++w) {
          float a2[N];
#pragma unroll
          for (int i = 0; i < N; ++i) a2[i] = sh[w][lane][2 + i];
          join<N>(m, l, acc, sh[w][lane][0], sh[w][lane][1], a2);
        }
    }
    if (lane < span && t.live) finish_forward<T, LPH, N>(p, t, m, l, acc);
  };
  int turn = 0;
  for (uint64_t left = small; left; left &= left - 1)
    if (turn++ % kWavesPerBlock == wave) join_row(__builtin_ctzll(left), false);
  for (uint64_t left = found & ~small; left; left &= left - 1) join_row(__builtin_ctzll(left), true);
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

template <typename T, int LPH, int N>
__device__ __forceinline__ void finish_rows(const AttnArgs &p, const Task &t, float m, float r, float d0, float rest,
                                            float (&a)[N], const float (&b)[N]) {
  if (t.d0 == 0) p.stats4[t.row * p.heads + t.head] = f32x4{m, r, d0 + rest, 0.0f};
  if (!p.o0) return;
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = (kCorrected<T> ? fmaf(-rest, b[i], a[i]) : a[i]) * p.scale;
  store_piece<T, LPH == 0>((T *)p.o0 + t.row * p.o0_row + t.head * p.o0_head + t.d0, p.dim, a);
}

// What a row's lanes hold of it in the row pass.
template <typename T, int LPH>
__device__ __forceinline__ typename Piece<T>::raw load_row(const AttnArgs &p, const Task &t, float &m, float &r, float &d0) {
  const typename Piece<T>::raw g = load_own<T, LPH>(p, t, p.dout, p.dout_row, p.dout_head);
  const typename Piece<T>::raw o = load_own<T, LPH>(p, t, p.out, p.out_row, p.out_head);
  const f32x2 st = load_at<f32x2>(at_or_zeros((Address)(p.stats + (t.row * p.heads + t.head) * 2), t.live));
  m = st[0];
  r = st[1];
  d0 = group_sum<LPH>(dot_piece<T>(g, o));
  return g;
}

template <typename T, int LPH, bool SHIFTS, bool RAGGED>
__global__ __launch_bounds__(kBlock, (kWaves<LPH, SHIFTS>)) void attention_backward_rows_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N;
  typedef typename Piece<T>::raw raw;
  __shared__ float sh[2 * N + 1][kWave];
  Task t;
  if (!find_task<T, LPH>(p, p.heads, t)) return;
  const int kv = t.head / p.group;
  float acc[N] = {}, low[N] = {}, m, r, d0, rest = 0.0f;
  const raw q = load_own<T, LPH>(p, t, p.q, p.q_row, p.q_head), g = load_row<T, LPH>(p, t, m, r, d0);
  const Address kb = (Address)((const T *)p.k + kv * p.k_head + t.d0), vb = (Address)((const T *)p.v + kv * p.v_head + t.d0);
  if (!kCorrected<T> && !p.o0) t.count = 0;        // delta alone is asked for
  if (t.count) {
    Edges<SHIFTS, kBackwardEdges> edges;
    edges.begin(p, t, [&](int u) { return t.edge + u * t.edges; });
    for (uint32_t x = t.edge; edges.more(); x += kBackwardEdges * t.edges) {
      raw k[kBackwardEdges], v[kBackwardEdges];
      float shift[kBackwardEdges];
      bool on[kBackwardEdges];
#pragma unroll
      for (int u = 0; u < kBackwardEdges; ++u) {
        on[u] = edges.next[u].on();
        shift[u] = edges.next[u].shift;
        k[u] = load_piece<T, LPH == 0>(at_or_zeros(row_at(kb, edges.next[u].col, p.k_bytes), on[u] && t.live), p.dim);
        v[u] = load_piece<T, LPH == 0>(at_or_zeros(row_at(vb, edges.next[u].col, p.v_bytes), on[u] && t.live), p.dim);
      }
      edges.advance(p, t, [&](int u) { return x + (edges.ahead * kBackwardEdges + u) * t.edges; });
      read_ahead_fence();
#pragma unroll
      for (int u = 0; u < kBackwardEdges; ++u) {
        const f32x2 sd = head_dots<T, LPH, RAGGED>(q, k[u], g, v[u], t.skip, p.dim);
        const float s = sd[0], d = sd[1];
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
  }
  for (int at = 1; at < t.side; at <<= 1) {
    const int off = ((LPH ? LPH : 1) * at) << p.heads_log2;
    rest += __shfl_xor(rest, off, kWave);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      acc[i] += __shfl_xor(acc[i], off, kWave);
      if constexpr (kCorrected<T>) low[i] += __shfl_xor(low[i], off, kWave);
    }
  }
  if (t.whole) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & (kWave - 1);
    for (int w = 1; w < kWavesPerBlock; ++w) {
      if (wave == w) {
        sh[0][lane] = rest;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sh[1 + i][lane] = acc[i];
          sh[1 + N + i][lane] = low[i];
        }
      }
      __syncthreads();
      if (wave == 0) {
        rest += sh[0][lane];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          acc[i] += sh[1 + i][lane];
          low[i] += sh[1 + N + i][lane];
        }
      }
      __syncthreads();
    }
    if (wave != 0) return;
  }
  if (!kCorrected<T>) rest = 0.0f;
  if (!t.first || !t.live) return;
  if (r == 0.0f) d0 = rest = 0.0f;   // a row of zeros hands nothing on, whatever its gradient holds
  if (t.piece >= 0) {
    float *part = p.part + t.piece * p.part_floats + (int64_t)t.head * (2 * kPartWide<T, LPH> + 4);
    store_floats<N>(part + t.d0, acc);
    store_floats<N>(part + kPartWide<T, LPH> + t.d0, low);
    if (t.d0 == 0) part[2 * kPartWide<T, LPH>] = rest;
    return;
  }
  finish_rows<T, LPH, N>(p, t, m, r, d0, rest, acc, low);
}

// Column pass: a row of the transpose is a column j of the pattern.  The lanes own
// the key heads; the edges of the column are walked once per query head that
// shares the key head, as count * group items.
template <typename T, int LPH, bool SHIFTS, bool RAGGED>
__global__ __launch_bounds__(kBlock, (kWaves<LPH, SHIFTS>)) void attention_backward_columns_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N;
  typedef typename Piece<T>::raw raw;
  __shared__ float sh[2 * N][kWave];
  Task t;
  if (!find_task<T, LPH>(p, p.kv_heads, t)) return;
  float dk[N] = {}, dv[N] = {};
  const raw k = load_own<T, LPH>(p, t, p.k, p.k_row, p.k_head), v = load_own<T, LPH>(p, t, p.v, p.v_row, p.v_head);
  const int head0 = t.head * p.group;
  const Address qb = (Address)((const T *)p.q + head0 * p.q_head + t.d0), gb = (Address)((const T *)p.dout + head0 * p.dout_head + t.d0),
                stb = (Address)(p.stats4 + head0);
  if (t.count) {
    const uint32_t group = p.group;
    // item x is edge x / group under query head x % group; `at`, `sub`: the next to read
    uint32_t at = t.edge / group, sub = t.edge - at * group;
    const uint32_t at_step = t.edges / group, sub_step = t.edges - at_step * group;
    constexpr int U = kBackwardEdges;
    Edges<SHIFTS, U> edges;
    uint32_t subs[2 * U];                          // query heads of the next edges and of the later ones
    const auto place = [&](int to) {
      const uint32_t x = at;
      subs[to] = sub;
      at += at_step;
      sub += sub_step;
      if (sub >= group) {
        sub -= group;
        ++at;
      }
      return x;
    };
    edges.begin(p, t, place);
    while (edges.more()) {
      raw q[kBackwardEdges], g[kBackwardEdges];
      f32x4 st[kBackwardEdges];
      float shift[kBackwardEdges];
      bool on[kBackwardEdges];
#pragma unroll
      for (int u = 0; u < kBackwardEdges; ++u) {
        on[u] = edges.next[u].on();
        shift[u] = edges.next[u].shift;
        const bool there = on[u] && t.live;
        const int32_t row = edges.next[u].col, h = subs[u];
        q[u] = load_piece<T, LPH == 0>(at_or_zeros(row_at(row_at(qb, row, p.q_bytes), h, p.q_head_bytes), there), p.dim);
        g[u] = load_piece<T, LPH == 0>(at_or_zeros(row_at(row_at(gb, row, p.dout_bytes), h, p.dout_head_bytes), there), p.dim);
        st[u] = load_at<f32x4>(at_or_zeros(row_at(stb, row, p.heads * 16) + h * 16, there));
      }
      if (SHIFTS) {
#pragma unroll
        for (int u = 0; u < U; ++u) subs[u] = subs[U + u];
      }
      edges.advance(p, t, [&](int u) { return place((edges.ahead - 1) * U + u); });
      read_ahead_fence();
#pragma unroll
      for (int u = 0; u < kBackwardEdges; ++u) {
        const f32x2 sd = head_dots<T, LPH, RAGGED>(k, q[u], v, g[u], t.skip, p.dim);
        const float s = sd[0], d = sd[1];
        const float w = on[u] ? exp_of(fmaf(s, p.scale, shift[u]) - st[u][0]) * st[u][1] : 0.0f;
        const float ds = on[u] ? w * (d - st[u][2]) : 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          dv[i] = fmaf(w, (float)g[u][i], dv[i]);
          dk[i] = fmaf(ds, (float)q[u][i], dk[i]);
        }
      }
    }
  }
  for (int at = 1; at < t.side; at <<= 1) {
    const int off = ((LPH ? LPH : 1) * at) << p.heads_log2;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      dk[i] += __shfl_xor(dk[i], off, kWave);
      dv[i] += __shfl_xor(dv[i], off, kWave);
    }
  }
  if (t.whole) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & (kWave - 1);
    for (int w = 1; w < kWavesPerBlock; ++w) {
      if (wave == w) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sh[i][lane] = dk[i];
          sh[N + i][lane] = dv[i];
        }
      }
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          dk[i] += sh[i][lane];
          dv[i] += sh[N + i][lane];
        }
      }
      __syncthreads();
    }
    if (wave != 0) return;
  }
  if (!t.first || !t.live) return;
  if (t.piece >= 0) {
    float *part = p.part + t.piece * p.part_floats + (int64_t)t.head * (2 * kPartWide<T, LPH> + 4);
    store_floats<N>(part + t.d0, dk);
    store_floats<N>(part + kPartWide<T, LPH> + t.d0, dv);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) dk[i] *= p.scale;
  store_piece<T, LPH == 0>((T *)p.o0 + t.row * p.o0_row + t.head * p.o0_head + t.d0, p.dim, dk);
  store_piece<T, LPH == 0>((T *)p.o1 + t.row * p.o1_row + t.head * p.o1_head + t.d0, p.dim, dv);
}

// Adds the pieces of cut rows in the backward passes: two vectors and a number a
// head (A, B and rest of the row pass; dk, dv and nothing of the column pass).
template <typename T, int LPH, bool COLUMNS>
__global__ __launch_bounds__(kBlock) void attention_backward_join_kernel(AttnArgs p) {
  constexpr int N = Piece<T>::N, L = LPH ? LPH : 1;
  const int span = L << p.heads_log2;        // lanes of a group
  __shared__ float sh[kWavesPerBlock][kWave][2 * N + 1];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  Task t;
  JoinTask j;
  int slot;
  place_lane<T, LPH>(p, COLUMNS ? p.kv_heads : p.heads, blockIdx.y, t, slot);
  const int head = t.live ? t.head : 0;      // lanes behind the last head read along
  int64_t rows, lasts;
  uint64_t small;
  const uint64_t found = find_joins(p, rows, lasts, small);
  const auto join_row = [&](int chunk, bool block) {
    const int groups = (block ? kBlock : kWave) / span, group = (block ? threadIdx.x : lane) / span;
    t.row = __shfl(rows, chunk, kWave);
    j.first = (int64_t)blockIdx.x * kJoinChunks + chunk;
    j.last = __shfl(lasts, chunk, kWave);
    float a[N] = {}, b[N] = {}, rest = 0.0f;
    for (int64_t c = j.first + group; c <= j.last; c += kJoinAhead * groups) {
      float a2[kJoinAhead][N], b2[kJoinAhead][N], rest2[kJoinAhead];
#pragma unroll
      for (int u = 0; u < kJoinAhead; ++u) {
        const float *part = j.part(p, c + u * groups) + (int64_t)head * (2 * kPartWide<T, LPH> + 4);
        load_floats<N>(part + t.d0, a2[u]);
        load_floats<N>(part + kPartWide<T, LPH> + t.d0, b2[u]);
        rest2[u] = COLUMNS ? 0.0f : part[2 * kPartWide<T, LPH>];
      }
#pragma unroll
      for (int u = 0; u < kJoinAhead; ++u)
        if (c + u * groups <= j.last) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            a[i] += a2[u][i];
            b[i] += b2[u][i];
          }
          rest += rest2[u];
        }
    }
    for (int off = span; off < kWave; off <<= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        a[i] += __shfl_xor(a[i], off, kWave);
        b[i] += __shfl_xor(b[i], off, kWave);
      }
      rest += __shfl_xor(rest, off, kWave);
    }
    float m = 0.0f, r = 0.0f, d0 = 0.0f;
    if (!COLUMNS && (!block || wave == 0)) load_row<T, LPH>(p, t, m, r, d0);
    if (block) {
      __syncthreads();
      if (lane < span) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          sh[wave][lane][i] = a[i];
          sh[wave][lane][N + i] = b[i];
        }
        sh[wave][lane][2 * N] = rest;
      }
      __syncthreads();
      if (wave != 0) return;
      if (lane < span)
#pragma unroll
        for (int w = 1; w < kWavesPerBlock; ++w) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            a[i] += sh[w][lane][i];
            b[i] += sh[w][lane][N + i];
          }
          rest += sh[w][lane][2 * N];
        }
    }
    if (lane >= span || !t.live) return;
    if constexpr (COLUMNS) {
#pragma unroll
      for (int i = 0; i < N; ++i) a[i] *= p.scale;
      store_piece<T, LPH == 0>((T *)p.o0 + t.row * p.o0_row + t.head * p.o0_head + t.d0, p.dim, a);
      store_piece<T, LPH == 0>((T *)p.o1 + t.row * p.o1_row + t.head * p.o1_head + t.d0, p.dim, b);
    } else {
      if (r == 0.0f) d0 = rest = 0.0f;
      finish_rows<T, LPH, N>(p, t, m, r, d0, rest, a, b);
    }
  };
  int turn = 0;
  for (uint64_t left = small; left; left &= left - 1)
    if (turn++ % kWavesPerBlock == wave) join_row(__builtin_ctzll(left), false);
  for (uint64_t left = found & ~small; left; left &= left - 1) join_row(__builtin_ctzll(left), true);
}

// ------------------------------------------------------------------ host side
enum { kForward = 0, kBackwardRows = 1, kBackwardColumns = 2 };

static int piece_elements(int dtype) { return dtype == GCNX_F32 ? 4 : 8; }

// 0: a head is shorter than a piece
static int lanes_per_head(int dtype, int dim) {
  const int n = piece_elements(dtype);
  return dim < n ? 0 : 1 << log2_ceil(ceil_div(dim, n));
}

static int64_t part_floats(int pass, int dtype, int heads, int kv_heads, int dim) {
  const int lph = lanes_per_head(dtype, dim);
  const int64_t wide = (int64_t)(lph ? lph : 1) * piece_elements(dtype);
  return pass == kForward ? heads * (wide + 4) : (pass == kBackwardRows ? heads : kv_heads) * (2 * wide + 4);
}

// Edges a wavefront takes of one row at most: a long row is the last to end where
// there are few rows, and pieces cost partial results where there are many.
// The forward pass with its join, us, at 64 / 128 / 256 / 512 (heads of 4 x 16, 8 on
// 2 x 64, 8 x 32, 8 x 32): 0.1 M edges 24 / 26 / 28 / 39, 0.9 M 177 / 181 / 220 / 256,
// 1 M 108 / 109 / 109 / 138, 8.5 M 1130 / 1096 / 1046 / 1057.
// Forward / backward at 128, 256, 512: 17.1 M (8 x 32 bf16) 2341/5315, 2299/5250,
// 2249/5158; (8 x 16 fp32) 2187/5137, 2184/5122, 2145/5033; 34.5 M (4 x 16 fp32)
// 2487/5935, 2444/5872, 2291/5554; 8.5 M (8 x 32 fp32) 2441/5195, 2401/5117, 2421/5228.
// Where rows average over 1024 pieces their joins are what takes long, and pieces get
// longer: 2^20 edges of 3 rows 133 / 111 / 95 / 115.
static int segment_of(int64_t nnz, int64_t n_rows) {
  int one = nnz <= (1 << 20) ? 64 : nnz <= (1 << 22) ? 128 : nnz <= (1 << 24) ? 256 : 512;
  while (one < 512 && n_rows * 1024 * one < nnz) one *= 2;
  return one;
}

// What becomes of rows longer than that.  Up to 8 times as long (if that is known)
// they get a workgroup each, whose wavefronts share the row and join in LDS; longer
// ones are cut into pieces and joined by a second launch (about 5 us).
enum RowCut { kNone, kWhole, kPieces };
static RowCut row_cut(int64_t nnz, int64_t n_rows, int64_t max_row_nnz) {
  const int64_t one = segment_of(nnz, n_rows);
  if (nnz <= one || (max_row_nnz > 0 && max_row_nnz <= one && nnz <= 0x7fffffff)) return kNone;
  return max_row_nnz > 0 && max_row_nnz <= 8 * one && nnz <= 0x7fffffff ? kWhole : kPieces;
}

static size_t part_bytes(const gcnx_attention *p, int64_t max_row_nnz, int pass) {
  const int64_t nnz = p->a->nnz, n_rows = pass == kBackwardColumns ? p->a->n_cols : p->a->n_rows;
  if (row_cut(nnz, n_rows, max_row_nnz) != kPieces) return 0;
  return align_up((size_t)(2 * ceil_div(nnz, segment_of(nnz, n_rows))) *
                      part_floats(pass, p->dtype, p->n_heads, p->n_kv_heads, p->head_dim) * sizeof(float), 256);
}

static size_t stats4_bytes(const gcnx_attention *p) {
  return align_up((size_t)p->a->n_rows * p->n_heads * 16, 256);
}

template <typename T, int LPH, bool SHIFTS, bool RAGGED>
static void launch_pass(int pass, const AttnArgs &p, dim3 grid, const AttnArgs &joined, dim3 joins, hipStream_t stream) {
  if (pass == kForward) {
    hipLaunchKernelGGL((attention_forward_kernel<T, LPH, SHIFTS, RAGGED>), grid, dim3(kBlock), 0, stream, p);
    if (p.part_floats) hipLaunchKernelGGL((attention_forward_join_kernel<T, LPH>), joins, dim3(kBlock), 0, stream, joined);
  } else if (pass == kBackwardRows) {
    hipLaunchKernelGGL((attention_backward_rows_kernel<T, LPH, SHIFTS, RAGGED>), grid, dim3(kBlock), 0, stream, p);
    if (p.part_floats) hipLaunchKernelGGL((attention_backward_join_kernel<T, LPH, false>), joins, dim3(kBlock), 0, stream, joined);
  } else {
    hipLaunchKernelGGL((attention_backward_columns_kernel<T, LPH, SHIFTS, RAGGED>), grid, dim3(kBlock), 0, stream, p);
    if (p.part_floats) hipLaunchKernelGGL((attention_backward_join_kernel<T, LPH, true>), joins, dim3(kBlock), 0, stream, joined);
  }
}

template <typename T, int LPH>
static int launch_lanes(int pass, AttnArgs p, hipStream_t stream) {
  const int heads = pass == kBackwardColumns ? p.kv_heads : p.heads;
  const int slots_log2 = log2_ceil(kWave / (LPH ? LPH : 1));
  const int heads_log2 = log2_ceil(heads);
  p.heads_log2 = heads_log2 < slots_log2 ? heads_log2 : slots_log2;
  const int spare = slots_log2 - p.heads_log2;
  // edges side by side, what is left takes further rows: as many edges as the average
  // row has, so that rows end soon, unless there are rows enough to fill the machine
  // (8 wavefronts a SIMD): then as many rounds as a lane has edges in
  // flight, so that few lanes idle.  (Cora, 4 edges in flight: 11 us against 18; 2^18
  // rows of 2: 285 against 160.)
  const int64_t items = ceil_div(p.nnz * (pass == kBackwardColumns ? p.group : 1), p.n_rows);
  int e = log2_ceil(items);
  if ((p.n_rows << (e < spare ? e : spare)) >> spare > 8 * 1024) e = log2_ceil(ceil_div(items, pass == kForward ? kForwardEdges : kBackwardEdges));
  p.edge_log2 = e < spare ? e : spare;
  p.row_log2 = spare - p.edge_log2;
  p.tiles = (int)ceil_div(heads, (int64_t)1 << p.heads_log2);
  p.tiles_log2 = p.tiles <= 8 && (p.tiles & (p.tiles - 1)) == 0 ? log2_ceil(p.tiles) : -1;
  int64_t blocks = ceil_div(p.n_pieces + ceil_div(p.n_rows, (int64_t)1 << p.row_log2), kWavesPerBlock);
  blocks = p.tiles_log2 >= 0 ? ceil_div(blocks, 8 >> p.tiles_log2) * 8 : blocks * p.tiles;
  const dim3 grid((unsigned)blocks);
  // few rows of many pieces: a workgroup per head instead of one for a tile of them
  AttnArgs joined = p;
  if (p.n_pieces / 2 / p.n_rows >= 16) joined.heads_log2 = 0;
  const int64_t join_blocks = ceil_div(p.n_pieces / 2, kJoinChunks), join_tiles = ceil_div(heads, (int64_t)1 << joined.heads_log2);
  GCNX_REQUIRE(blocks < (1ll << 32) / kBlock && join_blocks < (1ll << 32) / kBlock, GCNX_ERR_UNSUPPORTED,
               "attention: %lld rows, %lld nonzeros and %d heads are too many for one launch", (long long)p.n_rows, (long long)p.nnz, heads);
  const dim3 joins((unsigned)join_blocks, (unsigned)join_tiles);
  // one lane's head is a piece, or shorter; several lanes' may be a multiple of one
  const bool shifts = p.val || p.mask, ragged = LPH == 0 || p.dim % Piece<T>::N != 0;
  if constexpr (LPH != 1)
    if (ragged) {
      if (shifts) launch_pass<T, LPH, true, true>(pass, p, grid, joined, joins, stream);
      else launch_pass<T, LPH, false, true>(pass, p, grid, joined, joins, stream);
    }
  if constexpr (LPH != 0)
    if (!ragged) {
      if (shifts) launch_pass<T, LPH, true, false>(pass, p, grid, joined, joins, stream);
      else launch_pass<T, LPH, false, false>(pass, p, grid, joined, joins, stream);
    }
  GCNX_CHECK_LAUNCH();
  return GCNX_OK;
}

template <typename T>
static int launch_type(int pass, int lph, const AttnArgs &p, hipStream_t stream) {
  switch (lph) {
    case 0: return launch_lanes<T, 0>(pass, p, stream);
    case 1: return launch_lanes<T, 1>(pass, p, stream);
    case 2: return launch_lanes<T, 2>(pass, p, stream);
    case 4: return launch_lanes<T, 4>(pass, p, stream);
    case 8: return launch_lanes<T, 8>(pass, p, stream);
    case 16: return launch_lanes<T, 16>(pass, p, stream);
    case 32: return launch_lanes<T, 32>(pass, p, stream);
    default:
      if constexpr (Piece<T>::N == 4) return launch_lanes<T, 64>(pass, p, stream);
      else return GCNX_ERR_UNSUPPORTED;
  }
}

static int launch(int pass, int dtype, const AttnArgs &p, hipStream_t stream) {
  if (p.n_rows == 0) return GCNX_OK;
  const int lph = lanes_per_head(dtype, p.dim);
  return dtype == GCNX_F32 ? launch_type<float>(pass, lph, p, stream)
         : dtype == GCNX_BF16 ? launch_type<__bf16>(pass, lph, p, stream) : launch_type<_Float16>(pass, lph, p, stream);
}

// gathered rows are addressed by 32-bit byte strides
static bool stride_ok(int64_t elements) { return elements >= 0 && elements < (1ll << 30); }

static int check(const gcnx_attention *p) {
  GCNX_REQUIRE(p && p->a, GCNX_ERR_INVALID_ARG, "attention: null argument");
  GCNX_REQUIRE(p->dtype == GCNX_F32 || p->dtype == GCNX_BF16 || p->dtype == GCNX_F16, GCNX_ERR_UNSUPPORTED,
               "attention: dtype %d", p->dtype);
  GCNX_REQUIRE(p->head_dim >= 1 && p->head_dim <= 256, GCNX_ERR_UNSUPPORTED, "attention: head_dim %d outside 1..256",
               p->head_dim);
  GCNX_REQUIRE(p->n_kv_heads >= 1 && p->n_heads >= 1 && p->n_heads % p->n_kv_heads == 0 && p->n_heads <= 65535,
               GCNX_ERR_INVALID_ARG, "attention: %d query heads over %d key heads", p->n_heads, p->n_kv_heads);
  GCNX_REQUIRE(p->a->n_rows >= 0 && p->a->n_cols >= 0 && p->a->nnz >= 0 && p->a->n_rows < 2147483647 &&
                   p->a->n_cols < 2147483647, GCNX_ERR_INVALID_ARG, "attention: bad matrix size");
  GCNX_REQUIRE((p->a->n_rows == 0 || p->a->row_ptr) && (p->a->nnz == 0 || p->a->col_idx), GCNX_ERR_INVALID_ARG,
               "attention: null matrix array");
  GCNX_REQUIRE(p->a->nnz == 0 || (p->a->n_rows > 0 && p->a->n_cols > 0), GCNX_ERR_INVALID_ARG, "attention: nonzeros in an empty matrix");
  GCNX_REQUIRE(!p->use_values || p->a->nnz == 0 || p->a->val, GCNX_ERR_INVALID_ARG, "attention: values asked for, none given");
  GCNX_REQUIRE((p->a->n_rows == 0 || p->q) && (p->a->n_cols == 0 || (p->k && p->v)), GCNX_ERR_INVALID_ARG,
               "attention: null operand");
  GCNX_REQUIRE(stride_ok(p->q_row) && stride_ok(p->q_head) && stride_ok(p->k_row) && stride_ok(p->k_head) &&
                   stride_ok(p->v_row) && stride_ok(p->v_head), GCNX_ERR_INVALID_ARG, "attention: a stride outside 0..2^30 - 1");
  return GCNX_OK;
}

static AttnArgs common_args(const gcnx_attention *p) {
  AttnArgs g = {};
  g.q = p->q; g.q_row = p->q_row; g.q_head = p->q_head;
  g.k = p->k; g.k_row = p->k_row; g.k_head = p->k_head;
  g.v = p->v; g.v_row = p->v_row; g.v_head = p->v_head;
  const int64_t size = p->dtype == GCNX_F32 ? 4 : 2;
  g.q_bytes = (uint32_t)(p->q_row * size);
  g.q_head_bytes = (uint32_t)(p->q_head * size);
  g.k_bytes = (uint32_t)(p->k_row * size);
  g.v_bytes = (uint32_t)(p->v_row * size);
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
  g.segment = segment_of(a->nnz, a->n_rows);
  const RowCut cut = row_cut(a->nnz, a->n_rows, max_row_nnz);
  g.whole = cut == kWhole;
  g.n_pieces = cut == kNone ? 0 : ceil_div(a->nnz, g.segment) * (g.whole ? kWavesPerBlock : 2);
  g.part_floats = cut == kPieces ? part_floats(pass, p->dtype, p->n_heads, p->n_kv_heads, p->head_dim) : 0;
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
  GCNX_REQUIRE(out && stride_ok(out_row) && stride_ok(out_head) && ((uintptr_t)stats & 7) == 0 && ((uintptr_t)ws & 15) == 0,
               GCNX_ERR_INVALID_ARG, "attention: bad output, or stats or workspace not aligned");
  const size_t need = part_bytes(p, p->max_row_nnz, kForward);
  GCNX_REQUIRE(need == 0 || (ws && ws_bytes >= need), GCNX_ERR_WORKSPACE, "attention: workspace of %zu bytes needed, %zu given",
               need, ws_bytes);
  GCNX_REQUIRE(row_cut(p->a->nnz, p->a->n_rows, p->max_row_nnz) == kNone || chunk_row, GCNX_ERR_INVALID_ARG, "attention: chunk table needed");
  AttnArgs g = common_args(p);
  set_pattern(g, p, p->a, chunk_row, p->mask_index, p->max_row_nnz, kForward, (float *)ws);
  g.o0 = out; g.o0_row = out_row; g.o0_head = out_head;
  g.stats = stats;
  return launch(kForward, p->dtype, g, as_stream(stream));
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
  // the nonzeros have one order in the matrix and another in the transpose
  GCNX_REQUIRE(!p->edge_mask || at->nnz == 0 || p->mask_index || t_mask_index, GCNX_ERR_INVALID_ARG,
               "attention: the mask needs its index in the matrix, or in the transpose, or in both");
  GCNX_REQUIRE(p->a->n_rows == 0 || (out && dout && stats && stride_ok(out_row) && stride_ok(out_head) && stride_ok(dout_row) && stride_ok(dout_head)),
               GCNX_ERR_INVALID_ARG, "attention: bad output or gradient of it");
  GCNX_REQUIRE(((uintptr_t)stats & 7) == 0 && ((uintptr_t)ws & 15) == 0, GCNX_ERR_INVALID_ARG, "attention: stats or workspace not aligned");
  // gradients of no rows, or of no columns, are empty tensors, whose address may be null
  GCNX_REQUIRE((dk == nullptr) == (dv == nullptr) && (dq || dk || p->a->n_rows == 0 || p->a->n_cols == 0),
               GCNX_ERR_INVALID_ARG, "attention: dq, or dk and dv, or all three");
  if (!dq && !dk) return GCNX_OK;
  const size_t need = gcnx_attention_backward_workspace_bytes(p, t_max_row_nnz);
  GCNX_REQUIRE(need == 0 || (ws && ws_bytes >= need), GCNX_ERR_WORKSPACE,
               "attention: workspace of %zu bytes needed, %zu given", need, ws_bytes);
  GCNX_REQUIRE((row_cut(p->a->nnz, p->a->n_rows, p->max_row_nnz) == kNone || chunk_row) &&
                   (row_cut(p->a->nnz, p->a->n_cols, t_max_row_nnz) == kNone || t_chunk_row), GCNX_ERR_INVALID_ARG,
               "attention: chunk table needed");
  const int64_t hd = (int64_t)p->n_heads * p->head_dim, kd = (int64_t)p->n_kv_heads * p->head_dim;
  AttnArgs g = common_args(p);
  g.out = out; g.out_row = out_row; g.out_head = out_head;
  g.dout = dout; g.dout_row = dout_row; g.dout_head = dout_head;
  g.dout_bytes = (uint32_t)(dout_row * (p->dtype == GCNX_F32 ? 4 : 2));
  g.dout_head_bytes = (uint32_t)(dout_head * (p->dtype == GCNX_F32 ? 4 : 2));
  g.stats = const_cast<float *>(stats);
  g.stats4 = (f32x4 *)ws;
  float *part = (float *)((char *)ws + stats4_bytes(p));
  set_pattern(g, p, p->a, chunk_row, p->mask_index, p->max_row_nnz, kBackwardRows, part);
  g.o0 = dq; g.o0_row = hd; g.o0_head = p->head_dim;
  if (int rc = launch(kBackwardRows, p->dtype, g, as_stream(stream))) return rc;
  if (!dk) return GCNX_OK;
  set_pattern(g, p, at, t_chunk_row, t_mask_index, t_max_row_nnz, kBackwardColumns, part);
  g.o0 = dk; g.o0_row = kd; g.o0_head = p->head_dim;
  g.o1 = dv; g.o1_row = kd; g.o1_head = p->head_dim;
  return launch(kBackwardColumns, p->dtype, g, as_stream(stream));
}
