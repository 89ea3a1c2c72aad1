// One AdamW step over many tensors, its two moments held in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   w = w (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// 8 bits: blocks of 256 elements share a scale, a power of two (so that dividing by
// it is exact) that brings the block's largest value to 224..448; the values are
// e4m3 codes of m and of sqrt(v), whose range of 2^18 between the largest and the
// smallest step is one of 2^36 for v.  Two things keep the step sound where the
// codes are coarse (3 bits of fraction):
//   - rounding is by chance, floor(x / step + u) with u uniform in [0, 1): b2 = 0.999
//     moves v by a thousandth a step, which rounding to the nearest would lose for
//     good; the expected code is the value;
//   - sqrt(v) > 0 never becomes 0: m over eps alone would throw the weight away.
// u comes from Philox4x32-10 of (seed; element / 4, t), 16 bits for each of m and v:
// the same state on any launch geometry.  An element that is not finite keeps a NaN
// code and leaves its block's scale to the others.  Arithmetic is fp32, one rounding
// an operation (no contraction), so that the codes are those of the formulas above
// computed operation by operation.
//
// Bound by memory: 28 bytes an element with fp32 weights, gradients and state, 12 with
// fp32 weights, bf16 gradients and 8-bit state (scales are 1/32 byte each).  A
// wavefront takes tiles of 256 elements, 4 a lane, all loads of its tiles before the
// arithmetic; a block's largest values are found by exchanges within the wavefront.
// All tensors (64 a launch) are one launch: their addresses travel in the kernel's
// arguments, so gradients may move from step to step and nothing is uploaded.
#include "gcnx_common.h"
#include "gcnx_philox.h"
#include "gcnx_piece.h"

#include <math.h>

namespace gcnx {

constexpr int kTile = GCNX_ADAMW_BLOCK;       // elements that share a scale: 4 a lane
constexpr int kAdamTensors = 64;              // tensors a launch

struct AdamTable {
  void *w[kAdamTensors];
  const void *g[kAdamTensors];
  int64_t n[kAdamTensors];
  int64_t base[kAdamTensors];                 // of the tensor's state, a multiple of kTile
  float keep[kAdamTensors];                   // 1 - lr * decay
  uint32_t first[kAdamTensors + 1];           // first workgroup
  int32_t count;
};

struct AdamArgs {
  void *m, *v;
  float *m_scale, *v_scale;
  float b1, c1, b2, c2, eps;
  float step, root;                           // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  const float *t_terms;                       // those two from device memory, or NULL
  const uint64_t *t_dev;                      // and t
  uint64_t t, seed;
};

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x1;

template <typename T>
__device__ __forceinline__ f32x4 load4(const T *p, int64_t left) {
  typedef T four __attribute__((ext_vector_type(4)));
  typedef four anywhere __attribute__((aligned(sizeof(T))));
  f32x4 f = {0.0f, 0.0f, 0.0f, 0.0f};
  if (left >= 4) {
    const four x = *reinterpret_cast<const anywhere *>(p);
    f = f32x4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
  } else {
    for (int i = 0; i < 3; ++i)
      if (i < left) f[i] = (float)p[i];
  }
  return f;
}

template <typename T>
__device__ __forceinline__ void store4(T *p, int64_t left, const f32x4 &f) {
  typedef T four __attribute__((ext_vector_type(4)));
  typedef four anywhere __attribute__((aligned(sizeof(T))));
  if (left >= 4) {
    *reinterpret_cast<anywhere *>(p) = four{(T)f[0], (T)f[1], (T)f[2], (T)f[3]};
  } else {
    for (int i = 0; i < 3; ++i)
      if (i < left) p[i] = (T)f[i];
  }
}

__device__ __forceinline__ float wave_max(float v) {
#define GCNX_DPP(ctrl) __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), ctrl, 0xF, 0xF, true))
  v = fmaxf(v, GCNX_DPP(0xB1));
  v = fmaxf(v, GCNX_DPP(0x4E));
  v = fmaxf(v, GCNX_DPP(0x141));
  v = fmaxf(v, GCNX_DPP(0x140));
#undef GCNX_DPP
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}

// 2^e and its inverse, -126 <= e <= 126.
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// The exponent of the scale of a block whose largest finite value is `top`: the
// smallest, not below -100, with top <= 448 * 2^e.  A block of zeros has -9.
__device__ __forceinline__ int scale_exponent(float top) {
  const int bits = __float_as_int(top);
  const int e = (bits >> 23) - 126 - 9 + ((bits & 0x7fffff) > 0x600000);
  return top == 0.0f ? -9 : e < -100 ? -100 : e;
}

// |x| (already divided by the scale) on the e4m3 grid, rounded by u; NaN if x is not finite.
__device__ __forceinline__ float to_grid(float x, float u) {
  const int e = max(__float_as_int(x) >> 23, 127 - 6);
  const float q = floorf(x * __int_as_float((127 + 3 + 127 - e) << 23) + u) * __int_as_float((e - 3) << 23);
  return x < 1e30f ? fminf(q, 448.0f) : __builtin_nanf("");
}

__device__ __forceinline__ uint32_t pack_codes(const f32x4 &f) {
  uint32_t r = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], r, true);
}

__device__ __forceinline__ f32x4 unpack_codes(uint32_t c) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
  return f32x4{lo[0], lo[1], hi[0], hi[1]};
}

template <typename W, typename G, bool EIGHT, int TILES>
__global__ __launch_bounds__(kBlock) void adamw_kernel(AdamTable tab, AdamArgs p) {
#pragma clang fp contract(off)
  int lo = 0, hi = tab.count;                // the tensor of this workgroup
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const int64_t n = tab.n[lo], tile0 = ((int64_t)(blockIdx.x - tab.first[lo]) * kWavesPerBlock + (threadIdx.x >> 6)) * TILES;
  if (tile0 * kTile >= n) return;
  const int lane = threadIdx.x & (kWave - 1);
  W *w = (W *)tab.w[lo];
  const G *g = (const G *)tab.g[lo];
  const int64_t base = tab.base[lo];
  const float keep = tab.keep[lo];
  const float step = p.t_terms ? p.t_terms[0] : p.step, inv_root = p.t_terms ? p.t_terms[1] : p.root;
  const int64_t tiles = min((int64_t)TILES, (n - tile0 * kTile + kTile - 1) / kTile);
  f32x4 wv[TILES], gv[TILES], mv[TILES], vv[TILES];
  uint32_t mc[TILES], vc[TILES];
  float ms[TILES], vs[TILES];
#pragma unroll
  for (int k = 0; k < TILES; ++k) {
    const int64_t tile = k < tiles ? tile0 + k : tile0, at = tile * kTile + lane * 4;   // past the end: the first again, unused
    wv[k] = load4<W>(w + at, n - at);
    gv[k] = load4<G>(g + at, n - at);
    if constexpr (EIGHT) {
      mc[k] = *reinterpret_cast<const uint32_t *>((const uint8_t *)p.m + base + at);
      vc[k] = *reinterpret_cast<const uint32_t *>((const uint8_t *)p.v + base + at);
      ms[k] = p.m_scale[base / kTile + tile];
      vs[k] = p.v_scale[base / kTile + tile];
    } else {
      mv[k] = *reinterpret_cast<const f32x4 *>((const float *)p.m + base + at);
      vv[k] = *reinterpret_cast<const f32x4 *>((const float *)p.v + base + at);
    }
  }
#pragma unroll
  for (int k = 0; k < TILES; ++k) {
    if (k >= tiles) break;
    const int64_t tile = tile0 + k, at = tile * kTile + lane * 4;
    f32x4 m, v, root;
    if constexpr (EIGHT) {
      m = unpack_codes(mc[k]);
      v = unpack_codes(vc[k]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] *= ms[k];
        v[i] *= vs[k];
        v[i] *= v[i];
      }
    } else {
      m = mv[k];
      v = vv[k];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float gi = gv[k][i];
      m[i] = m[i] * p.b1 + gi * p.c1;
      v[i] = v[i] * p.b2 + (gi * gi) * p.c2;
      root[i] = sqrtf(v[i]);
      wv[k][i] = wv[k][i] * keep - m[i] * __builtin_amdgcn_rcpf(root[i] * inv_root + p.eps) * step;
    }
    store4<W>(w + at, n - at, wv[k]);
    if constexpr (EIGHT) {
      float top_m = 0.0f, top_v = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = fabsf(m[i]);
        top_m = fmaxf(top_m, a < 3e38f ? a : 0.0f);
        top_v = fmaxf(top_v, root[i] < 3e38f ? root[i] : 0.0f);
      }
      const int em = scale_exponent(wave_max(top_m)), ev = scale_exponent(wave_max(top_v));
      const float im = power_of_two(-em), iv = power_of_two(-ev);
      const philox4 chance = philox4x32_10((uint64_t)(base + at) >> 2, p.t_dev ? *p.t_dev : p.t, p.seed);
      f32x4 mq, vq;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float um = (float)(chance.v[i] & 0xffffu) * 0x1p-16f, uv = (float)(chance.v[i] >> 16) * 0x1p-16f;
        mq[i] = copysignf(to_grid(fabsf(m[i]) * im, um), m[i]);
        vq[i] = to_grid(root[i] * iv, uv);
        if (root[i] > 0.0f) vq[i] = vq[i] < 0x1p-9f ? 0x1p-9f : vq[i];
      }
      *reinterpret_cast<uint32_t *>((uint8_t *)p.m + base + at) = pack_codes(mq);
      *reinterpret_cast<uint32_t *>((uint8_t *)p.v + base + at) = pack_codes(vq);
      if (lane == 0) {
        p.m_scale[base / kTile + tile] = power_of_two(em);
        p.v_scale[base / kTile + tile] = power_of_two(ev);
      }
    } else {
      *reinterpret_cast<f32x4 *>((float *)p.m + base + at) = m;
      *reinterpret_cast<f32x4 *>((float *)p.v + base + at) = v;
    }
  }
}

// The two terms of step t, t being counted on the device.
__global__ void adamw_terms_kernel(const uint64_t *t_dev, double lr, double b1, double b2, float *terms) {
  const double t = (double)*t_dev;
  terms[0] = (float)(lr / (1.0 - pow(b1, t)));
  terms[1] = (float)(1.0 / sqrt(1.0 - pow(b2, t)));
}

template <typename W, typename G>
static void launch_adamw(bool eight, bool deep, unsigned blocks, const AdamTable &tab, const AdamArgs &p, hipStream_t stream) {
  if (eight) {
    if (deep) hipLaunchKernelGGL((adamw_kernel<W, G, true, 4>), dim3(blocks), dim3(kBlock), 0, stream, tab, p);
    else hipLaunchKernelGGL((adamw_kernel<W, G, true, 1>), dim3(blocks), dim3(kBlock), 0, stream, tab, p);
  } else {
    if (deep) hipLaunchKernelGGL((adamw_kernel<W, G, false, 4>), dim3(blocks), dim3(kBlock), 0, stream, tab, p);
    else hipLaunchKernelGGL((adamw_kernel<W, G, false, 1>), dim3(blocks), dim3(kBlock), 0, stream, tab, p);
  }
}

template <typename W>
static void launch_adamw(int g, bool eight, bool deep, unsigned blocks, const AdamTable &tab, const AdamArgs &p, hipStream_t stream) {
  if (g == GCNX_F32) launch_adamw<W, float>(eight, deep, blocks, tab, p, stream);
  else if (g == GCNX_BF16) launch_adamw<W, __bf16>(eight, deep, blocks, tab, p, stream);
  else launch_adamw<W, _Float16>(eight, deep, blocks, tab, p, stream);
}

}  // namespace gcnx

using namespace gcnx;

extern "C" int gcnx_adamw_step(const gcnx_adamw *q, int64_t n_tensors, const gcnx_adamw_tensor *h_tensors, void *ws, size_t ws_bytes,
                               void *stream) {
  GCNX_REQUIRE(q && n_tensors >= 0 && (n_tensors == 0 || h_tensors), GCNX_ERR_INVALID_ARG, "adamw: null argument");
  const auto known = [](int d) { return d == GCNX_F32 || d == GCNX_BF16 || d == GCNX_F16; };
  GCNX_REQUIRE(known(q->w_dtype) && known(q->g_dtype) && (q->state_bits == 32 || q->state_bits == 8), GCNX_ERR_UNSUPPORTED,
               "adamw: weight dtype %d, gradient dtype %d, %d-bit state", q->w_dtype, q->g_dtype, q->state_bits);
  GCNX_REQUIRE((q->t >= 1 || q->t_dev) && q->beta1 >= 0 && q->beta1 < 1 && q->beta2 >= 0 && q->beta2 < 1 && q->eps >= 0,
               GCNX_ERR_INVALID_ARG, "adamw: step count, betas or eps out of range");
  int64_t total = 0, live = 0;
  for (int64_t i = 0; i < n_tensors; ++i) {
    const gcnx_adamw_tensor &x = h_tensors[i];
    GCNX_REQUIRE(x.n >= 0 && x.state >= 0 && x.state % kTile == 0 && (x.n == 0 || (x.w && x.grad)), GCNX_ERR_INVALID_ARG,
                 "adamw: tensor %lld: null, negative size or a state offset that is no multiple of %d", (long long)i, kTile);
    total += x.n;
    live += x.n > 0;
  }
  if (live == 0) return GCNX_OK;
  const bool eight = q->state_bits == 8;
  GCNX_REQUIRE(q->exp_avg && q->exp_avg_sq && (!eight || (q->exp_avg_scale && q->exp_avg_sq_scale)) &&
                   (((uintptr_t)q->exp_avg | (uintptr_t)q->exp_avg_sq) & 15) == 0, GCNX_ERR_INVALID_ARG, "adamw: state null or not 16-byte aligned");
  AdamArgs p = {};
  p.m = q->exp_avg; p.v = q->exp_avg_sq;
  p.m_scale = q->exp_avg_scale; p.v_scale = q->exp_avg_sq_scale;
  p.b1 = (float)q->beta1; p.c1 = (float)(1.0 - q->beta1);
  p.b2 = (float)q->beta2; p.c2 = (float)(1.0 - q->beta2);
  p.eps = (float)q->eps;
  p.seed = q->seed;
  p.t = (uint64_t)q->t;
  if (q->t_dev) {
    GCNX_REQUIRE(ws && ws_bytes >= GCNX_ADAMW_WORKSPACE_BYTES, GCNX_ERR_WORKSPACE, "adamw: workspace of %d bytes needed, %zu given",
                 GCNX_ADAMW_WORKSPACE_BYTES, ws_bytes);
    p.t_dev = q->t_dev;
    p.t_terms = (const float *)ws;
    hipLaunchKernelGGL(adamw_terms_kernel, dim3(1), dim3(1), 0, as_stream(stream), q->t_dev, q->lr, q->beta1, q->beta2, (float *)ws);
    GCNX_CHECK_LAUNCH();
  } else {
    p.step = (float)(q->lr / (1.0 - pow(q->beta1, (double)q->t)));
    p.root = (float)(1.0 / sqrt(1.0 - pow(q->beta2, (double)q->t)));
  }
  // tiles a wavefront has in flight: 4 where they fill the machine (8 wavefronts a
  // SIMD), else 1, so that more of it takes part
  const bool deep = total / (4 * kTile) >= 8 * 1024;
  const int64_t per_block = (int64_t)kTile * kWavesPerBlock * (deep ? 4 : 1);
  for (int64_t i = 0; i < n_tensors;) {
    AdamTable tab = {};
    int64_t blocks = 0;
    for (; i < n_tensors && tab.count < kAdamTensors; ++i) {
      const gcnx_adamw_tensor &x = h_tensors[i];
      if (x.n == 0) continue;
      const int64_t more = ceil_div(x.n, per_block);
      GCNX_REQUIRE(more <= 0x7fffffff, GCNX_ERR_UNSUPPORTED, "adamw: tensor %lld is too large", (long long)i);
      if (blocks + more > 0x7fffffff) break;
      const int k = tab.count++;
      tab.w[k] = x.w;
      tab.g[k] = x.grad;
      tab.n[k] = x.n;
      tab.base[k] = x.state;
      tab.keep[k] = (float)(1.0 - q->lr * x.weight_decay);
      tab.first[k] = (uint32_t)blocks;
      blocks += more;
    }
    tab.first[tab.count] = (uint32_t)blocks;
    if (blocks == 0) continue;
    if (q->w_dtype == GCNX_F32) launch_adamw<float>(q->g_dtype, eight, deep, (unsigned)blocks, tab, p, as_stream(stream));
    else if (q->w_dtype == GCNX_BF16) launch_adamw<__bf16>(q->g_dtype, eight, deep, (unsigned)blocks, tab, p, as_stream(stream));
    else launch_adamw<_Float16>(q->g_dtype, eight, deep, (unsigned)blocks, tab, p, as_stream(stream));
    GCNX_CHECK_LAUNCH();
  }
  return GCNX_OK;
}
