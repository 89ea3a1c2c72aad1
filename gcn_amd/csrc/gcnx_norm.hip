// The norms around a block of a deep network, fused with the block's gate and
// residual scale, forward and backward.  Row by row of dim elements:
//
//   u = norm(z) * post      y = x + res * sigmoid(gate) * u      h = norm(y) * pre
//
// norm(a) = (a - mean) * inv with inv = 1 / sqrt(mean((a - mean)^2) + eps) and mean 0
// for the rms kind; every factor may be absent.  Backward, for the gradients dy, dh:
//
//   t  = dh pre          g  = dy + inv_y (t - mean(t) - y^ mean(t y^))      dx = g
//   du = g res sigmoid   dgate = g res u sigmoid (1 - sigmoid)
//   w  = du post         dz = inv_z (w - mean(w) - z^ mean(w z^))
//   dpre = sum dh y^     dres = sum g sigmoid u      dpost = sum du z^      over the rows
//
// with y^, z^ the normalised rows (the means of t and w only for the layer kind).
// The backward reads x and forms y again in 32 bits rather than reading the rounded
// y: the same bytes, and the sums over the rows keep their digits.
//
// Bound by memory: 5 row passes forward, 8 backward.  A row lives in registers, one
// 16-byte piece a lane, so every operand is read once; workgroups stay and walk the
// rows, the next row's pieces being loaded while the present one is summed, with the
// weights and the three column sums of the lane's elements in registers all along.
// 2^20 rows of 256, bf16: forward 0.54 ms (2.7 GB, 4.9 TB/s), backward 0.83 ms (4.3 GB,
// 5.2 TB/s), where a copy of 2 GiB moves 4.9; 19,717 rows of 500, fp16: forward 22 us
// (99 MB, 4.5 TB/s).
#include "gcnx_common.h"
#include "gcnx_piece.h"

namespace gcnx {

struct NormArgs {
  const void *x, *z, *gate, *dy, *dh;
  int64_t x_ld, z_ld, gate_ld, dy_ld, dh_ld;
  void *o0, *o1, *o2;                 // y, h; or dx, dz, dgate
  int64_t o0_ld, o1_ld, o2_ld;
  const float *post, *res, *pre;
  float *stats;                       // per row: mean and inverse of z, of y
  float *part;                        // [blocks][3][dim] sums of dpost, dres, dpre
  int64_t n;
  int32_t dim;
  float eps;
};

// The lane's place: a row is spread over TPR lanes (TPR 0: one lane, a row shorter
// than a piece).
struct Place {
  int32_t d0, skip, slot;
  bool live;
};

template <typename T, int TPR>
__device__ __forceinline__ Place place(int dim) {
  constexpr int W = TPR ? TPR : 1, N = Piece<T>::N;
  Place a;
  a.slot = TPR > kWave ? 0 : threadIdx.x / W;       // one row a workgroup there: the row is a scalar
  a.d0 = (threadIdx.x % W) * N;
  a.live = a.d0 < dim;
  a.skip = 0;
  if (TPR && a.d0 + N > dim) {
    a.skip = a.live ? a.d0 + N - dim : N;
    a.d0 = dim - N;
  }
  return a;
}

// Whether the lane counts element i of its piece.
template <int TPR>
__device__ __forceinline__ bool counts(const Place &a, int i, int dim) {
  return TPR ? i >= a.skip : i < dim;
}

// Sums of two numbers over the TPR lanes of a row, in every lane.  Rows wider than a
// wavefront go through LDS; calls take turns with the two halves of it, so that one
// barrier a call is enough.
template <int TPR>
__device__ __forceinline__ f32x2 row_sum(f32x2 v, float *sh, int &turn) {
  if constexpr (TPR <= kWave) {
    return f32x2{group_sum<TPR>(v[0]), group_sum<TPR>(v[1])};
  } else {
    constexpr int kWaves = TPR / kWave;
    v[0] = group_sum<kWave>(v[0]);
    v[1] = group_sum<kWave>(v[1]);
    f32x2 *half = reinterpret_cast<f32x2 *>(sh) + turn * kWaves;
    turn ^= 1;
    if ((threadIdx.x & (kWave - 1)) == 0) half[threadIdx.x / kWave] = v;
    __syncthreads();
    if constexpr (kWaves == 16) {
      // 1024 lanes have 128 registers each: 32 of them for the 16 pairs were spilled
      const f32x2 t = half[threadIdx.x % kWaves];
      return f32x2{group_sum<kWaves>(t[0]), group_sum<kWaves>(t[1])};
    } else {
      f32x2 t = half[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) t += half[w];
      return t;
    }
  }
}

// A workgroup has one row where it needs a barrier (its loop is then uniform).
template <int TPR>
constexpr int kNormBlock = TPR > kWave ? TPR : kBlock;
template <int TPR>
constexpr int kNormShared = TPR > kWave ? 4 * TPR / kWave : 1;

// Weights of the lane's elements; 1 where there are none, 0 in lanes behind the row.
template <typename T, int TPR>
__device__ __forceinline__ void load_weights(const float *w, const Place &a, int dim, float (&f)[Piece<T>::N]) {
#pragma unroll
  for (int i = 0; i < Piece<T>::N; ++i)
    f[i] = !a.live ? 0.0f : !w ? 1.0f : TPR ? w[a.d0 + i] : w[i < dim ? i : dim - 1];
}

template <typename T, int TPR>
__device__ __forceinline__ typename Piece<T>::raw load_row_piece(const void *base, int64_t ld, int64_t row, const Place &a, bool there, int dim) {
  return load_piece<T, TPR == 0>(at_or_zeros((Address)((const T *)base + row * ld + a.d0), there), dim);
}

// The normalised row from its elements: mean and inverse found on the way.
template <typename T, int TPR, bool LAYER>
__device__ __forceinline__ void normalise(const float (&v)[Piece<T>::N], const Place &a, int dim, float eps, float *sh, int &turn,
                                          float &mean, float &inv, float (&unit)[Piece<T>::N]) {
  constexpr int N = Piece<T>::N;
  mean = 0.0f;
  if (LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += counts<TPR>(a, i, dim) ? v[i] : 0.0f;
    mean = row_sum<TPR>(f32x2{s, 0.0f}, sh, turn)[0] / (float)dim;
  }
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    unit[i] = v[i] - mean;
    s += counts<TPR>(a, i, dim) ? unit[i] * unit[i] : 0.0f;
  }
  inv = 1.0f / sqrtf(row_sum<TPR>(f32x2{s, 0.0f}, sh, turn)[0] / (float)dim + eps);
#pragma unroll
  for (int i = 0; i < N; ++i) unit[i] *= inv;
}

// Off by (|g| + 6) 2^-24 of itself below 0 (where it is about e^g), by 2 ulp above:
// exp_of's product and the reciprocal (1 ulp) for the division.  It scales u, which is
// added to x: at g = -20 that is 1.3e-6 of a term of 2e-9 u.
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + exp_of(-g)); }

template <typename T, int TPR, bool LAYER>
__global__ __launch_bounds__(kNormBlock<TPR>) void norm_residual_kernel(NormArgs p) {
  constexpr int N = Piece<T>::N, kRows = kNormBlock<TPR> / (TPR ? TPR : 1);
  typedef typename Piece<T>::raw raw;
  __shared__ float sh[kNormShared<TPR>];
  int turn = 0;
  const Place a = place<T, TPR>(p.dim);
  float post[N], res[N], pre[N];
  load_weights<T, TPR>(p.post, a, p.dim, post);
  load_weights<T, TPR>(p.res, a, p.dim, res);
  load_weights<T, TPR>(p.pre, a, p.dim, pre);
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + a.slot;
  raw nx, nz, ng;
  auto read = [&](int64_t r) {
    const bool there = a.live && r < p.n;
    nx = load_row_piece<T, TPR>(p.x, p.x_ld, r, a, there, p.dim);
    nz = load_row_piece<T, TPR>(p.z, p.z_ld, r, a, there && p.z, p.dim);
    ng = load_row_piece<T, TPR>(p.gate, p.gate_ld, r, a, there && p.gate, p.dim);
  };
  read(row);
  for (; row < p.n; row += step) {
    const raw x = nx, z = nz, g = ng;
    read(row + step);
    read_ahead_fence();
    float y[N], unit[N], mean_z = 0.0f, inv_z = 0.0f, mean_y = 0.0f, inv_y = 0.0f;
    if (p.z) {
      float v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) unit[i] = v[i] = (float)z[i];
      if (p.post) normalise<T, TPR, LAYER>(v, a, p.dim, p.eps, sh, turn, mean_z, inv_z, unit);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float s = p.gate ? res[i] * sigmoid((float)g[i]) : res[i];
        y[i] = fmaf(s, unit[i] * post[i], (float)x[i]);
      }
      if (a.live) store_piece<T, TPR == 0>((T *)p.o0 + row * p.o0_ld + a.d0, p.dim, y);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = (float)x[i];
    }
    if (p.o1) {
      normalise<T, TPR, LAYER>(y, a, p.dim, p.eps, sh, turn, mean_y, inv_y, unit);
#pragma unroll
      for (int i = 0; i < N; ++i) unit[i] *= pre[i];
      if (a.live) store_piece<T, TPR == 0>((T *)p.o1 + row * p.o1_ld + a.d0, p.dim, unit);
    }
    if (p.stats && threadIdx.x % (TPR ? TPR : 1) == 0) *reinterpret_cast<f32x4 *>(p.stats + row * 4) = f32x4{mean_z, inv_z, mean_y, inv_y};
  }
}

// Backward through a norm: d, the gradient of the normalised row (times its weight),
// becomes the gradient of the row.
template <typename T, int TPR, bool LAYER>
__device__ __forceinline__ void normalise_backward(float (&d)[Piece<T>::N], const float (&unit)[Piece<T>::N], float inv, const Place &a,
                                                   int dim, float *sh, int &turn) {
  constexpr int N = Piece<T>::N;
  f32x2 s = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (counts<TPR>(a, i, dim)) {
      s[0] = fmaf(d[i], unit[i], s[0]);
      if (LAYER) s[1] += d[i];
    }
  s = row_sum<TPR>(s, sh, turn);
  const float along = s[0] / (float)dim, mean = LAYER ? s[1] / (float)dim : 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) d[i] = (d[i] - mean - unit[i] * along) * inv;
}

template <typename T, int TPR, bool LAYER>
__global__ __launch_bounds__(kNormBlock<TPR>) void norm_residual_backward_kernel(NormArgs p) {
  constexpr int N = Piece<T>::N, W = TPR ? TPR : 1, kRows = kNormBlock<TPR> / W;
  typedef typename Piece<T>::raw raw;
  __shared__ float sh[kNormShared<TPR>];
  __shared__ float col[kRows > 1 ? kWavesPerBlock : 1][kRows > 1 ? W * N : 1];
  int turn = 0;
  const Place a = place<T, TPR>(p.dim);
  float post[N], res[N], pre[N], dpost[N] = {}, dres[N] = {}, dpre[N] = {};
  load_weights<T, TPR>(p.post, a, p.dim, post);
  load_weights<T, TPR>(p.res, a, p.dim, res);
  load_weights<T, TPR>(p.pre, a, p.dim, pre);
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + a.slot;
  raw nx, nz, ng, ndy, ndh;
  f32x4 nst;
  auto read = [&](int64_t r) {
    const bool there = a.live && r < p.n;
    nx = load_row_piece<T, TPR>(p.x, p.x_ld, r, a, there, p.dim);
    nz = load_row_piece<T, TPR>(p.z, p.z_ld, r, a, there && p.z, p.dim);
    ng = load_row_piece<T, TPR>(p.gate, p.gate_ld, r, a, there && p.gate, p.dim);
    ndy = load_row_piece<T, TPR>(p.dy, p.dy_ld, r, a, there && p.dy, p.dim);
    ndh = load_row_piece<T, TPR>(p.dh, p.dh_ld, r, a, there && p.dh, p.dim);
    nst = load_at<f32x4>(at_or_zeros((Address)(p.stats + r * 4), r < p.n));
  };
  read(row);
  for (; row < p.n; row += step) {
    const raw x = nx, z = nz, gt = ng, dy = ndy, dh = ndh;
    const f32x4 st = nst;
    read(row + step);
    read_ahead_fence();
    float unit[N], u[N], sig[N], g[N], y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      g[i] = (float)dy[i];
      unit[i] = (float)z[i];
      if (p.post) unit[i] = (unit[i] - st[0]) * st[1];
      u[i] = unit[i] * post[i];
      sig[i] = p.gate ? sigmoid((float)gt[i]) : 1.0f;
      y[i] = p.z ? fmaf(res[i] * sig[i], u[i], (float)x[i]) : (float)x[i];
    }
    if (p.dh) {
      float t[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        y[i] = (y[i] - st[2]) * st[3];
        dpre[i] = fmaf((float)dh[i], y[i], dpre[i]);
        t[i] = (float)dh[i] * pre[i];
      }
      normalise_backward<T, TPR, LAYER>(t, y, st[3], a, p.dim, sh, turn);
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] += t[i];
    }
    if (a.live && p.o0) store_piece<T, TPR == 0>((T *)p.o0 + row * p.o0_ld + a.d0, p.dim, g);
    if (p.z) {
      float d[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float gs = g[i] * sig[i];
        dres[i] = fmaf(gs, u[i], dres[i]);
        d[i] = gs * res[i];
        y[i] = d[i] * u[i] * (1.0f - sig[i]);
      }
      if (a.live && p.o2) store_piece<T, TPR == 0>((T *)p.o2 + row * p.o2_ld + a.d0, p.dim, y);
      if (p.post) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          dpost[i] = fmaf(d[i], unit[i], dpost[i]);
          d[i] *= post[i];
        }
        normalise_backward<T, TPR, LAYER>(d, unit, st[1], a, p.dim, sh, turn);
      }
      if (a.live && p.o1) store_piece<T, TPR == 0>((T *)p.o1 + row * p.o1_ld + a.d0, p.dim, d);
    }
  }
  if (!p.part) return;
  // column sums of the workgroup: the rows side by side are added by exchanges in the
  // wavefront, then through LDS
  float *out = p.part + (int64_t)blockIdx.x * 3 * p.dim;
  auto finish = [&](const float (&sum)[N], float *to) {
    float total[N];
#pragma unroll
    for (int i = 0; i < N; ++i) total[i] = sum[i];
    if constexpr (kRows > 1) {
      for (int off = W; off < kWave; off <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) total[i] += __shfl_xor(total[i], off, kWave);
      const int share = threadIdx.x / kWave, at = threadIdx.x % W;
      __syncthreads();
      if ((threadIdx.x & (kWave - 1)) < W)
#pragma unroll
        for (int i = 0; i < N; ++i) col[share][at * N + i] = total[i];
      __syncthreads();
      if (a.slot == 0)
        for (int r = 1; r < kWavesPerBlock; ++r)
#pragma unroll
          for (int i = 0; i < N; ++i) total[i] += col[r][threadIdx.x * N + i];
    }
    if (a.slot == 0 && a.live)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (counts<TPR>(a, i, p.dim)) to[a.d0 + i] = total[i];
  };
  if (p.z && p.post) finish(dpost, out);
  if (p.z && p.res) finish(dres, out + p.dim);
  if (p.dh) finish(dpre, out + 2 * p.dim);
}

// out[which][d] = sum over the blocks: 16 columns and 16 shares of the blocks a
// workgroup, in a fixed order.
constexpr int kSumColumns = 16;
__global__ __launch_bounds__(kBlock) void norm_residual_columns_kernel(const float *__restrict__ part, int blocks, int dim, float *dpost,
                                                                       float *dres, float *dpre) {
  constexpr int kShares = kBlock / kSumColumns;
  __shared__ float sh[kShares][kSumColumns];
  const int c = threadIdx.x % kSumColumns, share = threadIdx.x / kSumColumns, which = blockIdx.y;
  float *out = which == 0 ? dpost : which == 1 ? dres : dpre;
  if (!out) return;
  const int d = blockIdx.x * kSumColumns + c;
  float s = 0.0f;
  if (d < dim) {
    const float *at = part + (int64_t)which * dim + d;
    int b = share;
    for (; b + 7 * kShares < blocks; b += 8 * kShares) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = at[(int64_t)(b + u * kShares) * 3 * dim];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
    for (; b < blocks; b += kShares) s += at[(int64_t)b * 3 * dim];
  }
  sh[share][c] = s;
  __syncthreads();
  if (share == 0 && d < dim) {
    for (int i = 1; i < kShares; ++i) s += sh[i][c];
    out[d] = s;
  }
}

// ------------------------------------------------------------------ host side
static int threads_per_row(int dtype, int dim) {
  const int n = dtype == GCNX_F32 ? 4 : 8;
  return dim < n ? 0 : 1 << log2_ceil(ceil_div(dim, n));
}

static int64_t rows_per_block(int tpr) { return tpr > kWave ? 1 : kBlock / (tpr ? tpr : 1); }

// Workgroups that stay: `deep` times 256 lanes a CU, in whole workgroups and at least
// one, fewer than the registers would hold (6 and 3 in 16 bits).  The backward pass
// writes a partial sum of the columns a workgroup; a CU with half a workgroup more than
// its neighbours ends last, and one without any idles.
// us forward / backward at 1, 2, 3, 4, 8 (rows x elements):
//   2^22 x 16, fp32     371/439  290/460  284/453  285/482  292/499   bf16  218/236  151/248  158/248  159/267  162/261
//   2^18 x 500, fp32    865/970  565/964  603/1005 608/1018 625/1025  bf16  421/422  290/466  291/490  298/514  309/500
//   2^20 x 256, fp32   1508/1740 1081/1719 1094/1689 1176/1785 1178/1795 bf16 763/818 531/839  546/890  582/1027 608/1094
//   2^17 x 1024, fp32   692/800  532/963  536/882  572/981  569/1038  bf16  438/516  291/444  285/456  281/487  283/492
// (1024 lanes a row, 2^15 x 4096 fp32: 64 x deep workgroups 523/1117, one a CU 494/800;
// 512 lanes, 2^15 x 4096 bf16: one and a half a CU 284/470, one 251/429.)
static int64_t norm_blocks(int64_t n, int tpr, int64_t deep) {
  const int64_t every = ceil_div(n, rows_per_block(tpr)), a_cu = deep * kBlock / (tpr > kWave ? tpr : kBlock);
  const int64_t most = 256 * (a_cu > 1 ? a_cu : 1);
  return every < most ? every : most;
}
constexpr int64_t kForwardDeep = 3, kBackwardDeep = 2;

template <typename T, bool LAYER>
static void launch_norm(bool backward, int tpr, int64_t blocks, const NormArgs &p, hipStream_t stream) {
#define GCNX_NORM(TPR)                                                                                            \
  case TPR:                                                                                                       \
    if (backward)                                                                                                 \
      hipLaunchKernelGGL((norm_residual_backward_kernel<T, TPR, LAYER>), dim3((unsigned)blocks),                  \
                         dim3(kNormBlock<TPR>), 0, stream, p);                                                    \
    else                                                                                                          \
      hipLaunchKernelGGL((norm_residual_kernel<T, TPR, LAYER>), dim3((unsigned)blocks), dim3(kNormBlock<TPR>), 0, \
                         stream, p);                                                                              \
    return;
  switch (tpr) {
    GCNX_NORM(0) GCNX_NORM(1) GCNX_NORM(2) GCNX_NORM(4) GCNX_NORM(8) GCNX_NORM(16) GCNX_NORM(32) GCNX_NORM(64)
    GCNX_NORM(128) GCNX_NORM(256) GCNX_NORM(512)
    default: break;
  }
  if constexpr (sizeof(T) == 4) switch (tpr) { GCNX_NORM(1024) }
#undef GCNX_NORM
}

static int launch(const gcnx_norm_residual *q, bool backward, int64_t blocks, const NormArgs &p, hipStream_t stream) {
  const int tpr = threads_per_row(q->dtype, q->dim);
  const bool layer = q->layer != 0;
  if (q->dtype == GCNX_F32) layer ? launch_norm<float, true>(backward, tpr, blocks, p, stream) : launch_norm<float, false>(backward, tpr, blocks, p, stream);
  else if (q->dtype == GCNX_BF16) layer ? launch_norm<__bf16, true>(backward, tpr, blocks, p, stream) : launch_norm<__bf16, false>(backward, tpr, blocks, p, stream);
  else layer ? launch_norm<_Float16, true>(backward, tpr, blocks, p, stream) : launch_norm<_Float16, false>(backward, tpr, blocks, p, stream);
  GCNX_CHECK_LAUNCH();
  return GCNX_OK;
}

static int check(const gcnx_norm_residual *p) {
  GCNX_REQUIRE(p, GCNX_ERR_INVALID_ARG, "norm_residual: null argument");
  GCNX_REQUIRE(p->dtype == GCNX_F32 || p->dtype == GCNX_BF16 || p->dtype == GCNX_F16, GCNX_ERR_UNSUPPORTED, "norm_residual: dtype %d", p->dtype);
  GCNX_REQUIRE(p->dim >= 1 && p->dim <= 4096, GCNX_ERR_UNSUPPORTED, "norm_residual: dim %d outside 1..4096", p->dim);
  GCNX_REQUIRE(p->n >= 0 && p->x_ld >= 0 && p->z_ld >= 0 && p->gate_ld >= 0, GCNX_ERR_INVALID_ARG, "norm_residual: negative size or stride");
  GCNX_REQUIRE(p->n == 0 || p->x, GCNX_ERR_INVALID_ARG, "norm_residual: null operand");
  GCNX_REQUIRE(p->z || (!p->gate && !p->post_weight && !p->res_scale), GCNX_ERR_INVALID_ARG,
               "norm_residual: gate, post_weight and res_scale belong to z");
  GCNX_REQUIRE(p->z || p->pre_weight, GCNX_ERR_INVALID_ARG, "norm_residual: neither z nor pre_weight: nothing to do");
  return GCNX_OK;
}

static NormArgs norm_args(const gcnx_norm_residual *q) {
  NormArgs p = {};
  p.x = q->x; p.x_ld = q->x_ld;
  p.z = q->z; p.z_ld = q->z_ld;
  p.gate = q->gate; p.gate_ld = q->gate_ld;
  p.post = q->post_weight; p.res = q->res_scale; p.pre = q->pre_weight;
  p.n = q->n;
  p.dim = q->dim;
  p.eps = q->eps;
  return p;
}

}  // namespace gcnx

using namespace gcnx;

extern "C" int gcnx_norm_residual_forward(const gcnx_norm_residual *q, void *y, int64_t y_ld, void *h, int64_t h_ld,
                                          float *stats, void *stream) {
  if (int rc = check(q)) return rc;
  if (q->n == 0) return GCNX_OK;
  GCNX_REQUIRE((!q->z || (y && y_ld >= q->dim)) && (!q->pre_weight || (h && h_ld >= q->dim)) && ((uintptr_t)stats & 15) == 0,
               GCNX_ERR_INVALID_ARG, "norm_residual: bad output");
  NormArgs p = norm_args(q);
  p.o0 = y; p.o0_ld = y_ld;
  p.o1 = q->pre_weight ? h : nullptr; p.o1_ld = h_ld;
  p.stats = stats;
  return launch(q, false, norm_blocks(q->n, threads_per_row(q->dtype, q->dim), kForwardDeep), p, as_stream(stream));
}

extern "C" size_t gcnx_norm_residual_backward_workspace_bytes(const gcnx_norm_residual *q) {
  if (check(q) != GCNX_OK || q->n == 0) return 0;
  return (size_t)norm_blocks(q->n, threads_per_row(q->dtype, q->dim), kBackwardDeep) * 3 * q->dim * sizeof(float);
}

extern "C" int gcnx_norm_residual_backward(const gcnx_norm_residual *q, const void *dy, int64_t dy_ld, const void *dh, int64_t dh_ld,
                                           const float *stats, void *dx, void *dz, void *dgate, float *dpost, float *dres,
                                           float *dpre, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check(q)) return rc;
  GCNX_REQUIRE((!dz || q->z) && (!dgate || q->gate) && (!dpost || q->post_weight) && (!dres || q->res_scale) && (!dpre || (q->pre_weight && dh)),
               GCNX_ERR_INVALID_ARG, "norm_residual: a gradient of an operand that is not there");
  GCNX_REQUIRE(!dh || q->pre_weight, GCNX_ERR_INVALID_ARG, "norm_residual: dh without pre_weight");
  const bool sums = dpost || dres || dpre;
  if (q->n == 0) {
    GCNX_REQUIRE(!sums, GCNX_ERR_INVALID_ARG, "norm_residual: sums over no rows");
    return GCNX_OK;
  }
  GCNX_REQUIRE(stats && ((uintptr_t)stats & 15) == 0 && dy_ld >= 0 && dh_ld >= 0, GCNX_ERR_INVALID_ARG, "norm_residual: bad stats or stride");
  const size_t need = sums ? gcnx_norm_residual_backward_workspace_bytes(q) : 0;
  GCNX_REQUIRE(need == 0 || (ws && ws_bytes >= need), GCNX_ERR_WORKSPACE, "norm_residual: workspace of %zu bytes needed, %zu given",
               need, ws_bytes);
  NormArgs p = norm_args(q);
  p.dy = dy; p.dy_ld = dy_ld;
  p.dh = dh; p.dh_ld = dh_ld;
  p.stats = const_cast<float *>(stats);
  p.o0 = dx; p.o1 = dz; p.o2 = dgate;
  p.o0_ld = p.o1_ld = p.o2_ld = q->dim;
  p.part = sums ? (float *)ws : nullptr;
  const int64_t blocks = norm_blocks(q->n, threads_per_row(q->dtype, q->dim), kBackwardDeep);
  if (int rc = launch(q, true, blocks, p, as_stream(stream))) return rc;
  if (!sums) return GCNX_OK;
  hipLaunchKernelGGL(norm_residual_columns_kernel, dim3((unsigned)ceil_div(q->dim, kSumColumns), 3), dim3(kBlock), 0, as_stream(stream),
                     (const float *)ws, (int)blocks, q->dim, dpost, dres, dpre);
  GCNX_CHECK_LAUNCH();
  return GCNX_OK;
}
