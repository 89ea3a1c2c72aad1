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
// computed operation by operation.  The one exception is the division of the step,
// which is the hardware's reciprocal (1 ulp) and a product: two more roundings of a
// term that is about lr, below the rounding of the weight that it changes, for a
// quarter of the division's instructions.
//
// Bound by memory: 28 bytes an element with fp32 weights, gradients and state, 14 with
// fp32 weights, bf16 gradients and 8-bit state (scales are 1/32 byte each).  A
// wavefront takes tiles of 256 elements, 4 a lane, all loads of its tiles before the
// arithmetic; a block's largest values are found by exchanges within the wavefront.
// All tensors (64 a launch) are one launch: their addresses travel in the kernel's
// arguments, so gradients may move from step to step and nothing is uploaded.
// 0.36 G elements in 32 bits: 1.75 ms (10.1 GB, 5.8 TB/s); 0.73 G elements with bf16
// gradients and 8-bit state: 1.75 to 1.9 ms (10.2 GB, 5.8 to 5.4 TB/s; the integer
// work of rounding is hidden just about).
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

template <bool STREAM, typename V, typename P>
__device__ __forceinline__ V load_as(const P *p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
  else return *reinterpret_cast<const V *>(p);
}
template <bool STREAM, typename V, typename P>
__device__ __forceinline__ void store_as(P *p, const V &v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<V *>(p));
  else *reinterpret_cast<V *>(p) = v;
}

// Four elements at p, `left` of them there.  FULL: all are, for the whole wavefront
// (a load under a condition is waited for before the next is issued).
template <bool FULL, bool STREAM, typename T>
__device__ __forceinline__ f32x4 load4(const T *p, int64_t left) {
  typedef T four __attribute__((ext_vector_type(4)));
  typedef four anywhere __attribute__((aligned(sizeof(T))));
  f32x4 f = {0.0f, 0.0f, 0.0f, 0.0f};
  if (FULL || left >= 4) {
    const anywhere x = load_as<STREAM, anywhere>(p);
    f = f32x4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
  } else {
    for (int i = 0; i < 3; ++i)
      if (i < left) f[i] = (float)p[i];
  }
  return f;
}

template <bool FULL, bool STREAM, typename T>
__device__ __forceinline__ void store4(T *p, int64_t left, const f32x4 &f) {
  typedef T four __attribute__((ext_vector_type(4)));
  typedef four anywhere __attribute__((aligned(sizeof(T))));
  if (FULL || left >= 4) {
    store_as<STREAM, anywhere>(p, anywhere{(T)f[0], (T)f[1], (T)f[2], (T)f[3]});
  } else {
    for (int i = 0; i < 3; ++i)
      if (i < left) p[i] = (T)f[i];
  }
}

// The largest over the wavefront, in a scalar register: shifts by 1, 2, 4, 8 lanes of
// a row of 16, then the last lane of each row to the rows behind it.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#define GCNX_STEP(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xF, false))
  GCNX_STEP(0x111, 0xF);
  GCNX_STEP(0x112, 0xF);
  GCNX_STEP(0x114, 0xF);
  GCNX_STEP(0x118, 0xF);
  GCNX_STEP(0x142, 0xA);
  GCNX_STEP(0x143, 0xC);
#undef GCNX_STEP
  return __builtin_amdgcn_readlane(v, kWave - 1);
}

constexpr uint32_t kSign = 0x80000000u, kInfinity = 0x7f800000u;

// 2^e, -126 <= e <= 127.
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The exponent of the scale of a block whose largest finite value has these bits: the
// smallest, not below -100, with value <= 448 * 2^e.  A block of zeros has -9.
__device__ __forceinline__ int scale_exponent(uint32_t top) {
  const int e = (int)(top >> 23) - 126 - 9 + ((top & 0x7fffff) > 0x600000);
  return top == 0 ? -9 : e < -100 ? -100 : e;
}

// The value of these bits (not negative, finite) over 2^e on the e4m3 grid, rounded
// by chance: floor(x / step + word / 2^16) * step with the step of x's binade, or the
// one of 2^-6 below.  Powers of two are built from the exponent bits; at most 448.
__device__ __forceinline__ float to_grid(uint32_t bits, int e, uint32_t word) {
  const uint32_t binade = max(bits & kInfinity, (uint32_t)(127 - 6 + e) << 23);       // 2^b, b the exponent of x or -6
  const float per_step = __uint_as_float(((uint32_t)(127 + 127 + 3) << 23) - binade);  // 2^(3 - b)
  const float step = __uint_as_float(binade - ((uint32_t)(3 + e) << 23));              // 2^(b - 3 - e)
  return floorf(fmaf((float)word, 0x1p-16f, __uint_as_float(bits) * per_step)) * step;
}

// sqrt, correctly rounded, of four numbers that are not negative.  One step from the
// reciprocal square root with exact residual is as good as the library's sequence of
// 16 instructions in half of them (every fraction and both parities of the exponent
// agree) unless the number is below 2^-100 or not finite; zero is.
__device__ __forceinline__ f32x4 root4(const f32x4 &x) {
  f32x4 r;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = __float_as_uint(x[i]);
    const float y = __builtin_amdgcn_rsqf(x[i]), s = x[i] * y;
    r[i] = b ? fmaf(fmaf(-s, s, x[i]), 0.5f * y, s) : 0.0f;
    odd = odd || (b && b - (27u << 23) >= kInfinity - (27u << 23));
  }
  if (__any(odd))
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = sqrtf(x[i]);
  return r;
}

__device__ __forceinline__ uint32_t pack_codes(const f32x4 &f) {
  uint32_t r = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], r, true);
}

__device__ __forceinline__ f32x4 unpack_codes(uint32_t c) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
  return f32x4{lo[0], lo[1], hi[0], hi[1]};
}

// What a wavefront has of one tensor.
template <typename W, typename G>
struct AdamSlice {
  W *w;
  const G *g;
  int64_t n, base, tile0;
  float keep;
};

// TILES tiles from tile0 on.  FULL: all of them are there, whole.
template <typename W, typename G, bool EIGHT, int TILES, bool STREAM, bool FULL>
__device__ __forceinline__ void adamw_tiles(const AdamArgs &p, const AdamSlice<W, G> &s) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & (kWave - 1);
  W *const w = s.w;
  const G *const g = s.g;
  const int64_t n = s.n, base = s.base, tile0 = s.tile0;
  const float step = p.t_terms ? p.t_terms[0] : p.step, inv_root = p.t_terms ? p.t_terms[1] : p.root;
  const int64_t tiles = FULL ? TILES : min((int64_t)TILES, (n - tile0 * kTile + kTile - 1) / kTile);
  f32x4 wv[TILES], gv[TILES], mv[TILES], vv[TILES];
  uint32_t mc[TILES], vc[TILES];
  float ms[TILES], vs[TILES];
#pragma unroll
  for (int k = 0; k < TILES; ++k) {
    const int64_t tile = k < tiles ? tile0 + k : tile0, at = tile * kTile + lane * 4;   // past the end: the first again, unused
    wv[k] = load4<FULL, STREAM, W>(w + at, n - at);
    gv[k] = load4<FULL, STREAM, G>(g + at, n - at);
    if constexpr (EIGHT) {
      mc[k] = load_as<STREAM, uint32_t>((const uint8_t *)p.m + base + at);
      vc[k] = load_as<STREAM, uint32_t>((const uint8_t *)p.v + base + at);
      ms[k] = p.m_scale[base / kTile + tile];
      vs[k] = p.v_scale[base / kTile + tile];
    } else {
      mv[k] = load_as<STREAM, f32x4>((const float *)p.m + base + at);
      vv[k] = load_as<STREAM, f32x4>((const float *)p.v + base + at);
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
    }
    root = root4(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wv[k][i] = wv[k][i] * s.keep - m[i] * __builtin_amdgcn_rcpf(root[i] * inv_root + p.eps) * step;
    }
    store4<FULL, STREAM, W>(w + at, n - at, wv[k]);
    if constexpr (EIGHT) {
      // not negative, so that bits compare as values do
      uint32_t bm[4], bv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bm[i] = __float_as_uint(m[i]) & ~kSign;
        bv[i] = __float_as_uint(root[i]) & ~kSign;
      }
      uint32_t top_m = wave_max(max(max(bm[0], bm[1]), max(bm[2], bm[3])));
      uint32_t top_v = wave_max(max(max(bv[0], bv[1]), max(bv[2], bv[3])));
      uint32_t bad_m = 0, bad_v = 0;             // elements that are not finite
      if (top_m >= kInfinity || top_v >= kInfinity) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (bm[i] >= kInfinity) { bad_m |= 1u << i; bm[i] = 0; }
          if (bv[i] >= kInfinity) { bad_v |= 1u << i; bv[i] = 0; }
        }
        top_m = wave_max(max(max(bm[0], bm[1]), max(bm[2], bm[3])));
        top_v = wave_max(max(max(bv[0], bv[1]), max(bv[2], bv[3])));
      }
      const int em = scale_exponent(top_m), ev = scale_exponent(top_v);
      const philox4 chance = philox4x32_10((uint64_t)(base + at) >> 2, p.t_dev ? *p.t_dev : p.t, p.seed);
      f32x4 mq, vq;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mq[i] = copysignf(to_grid(bm[i], em, chance.v[i] & 0xffffu), m[i]);
        vq[i] = fmaxf(to_grid(bv[i], ev, chance.v[i] >> 16), bv[i] ? 0x1p-9f : 0.0f);
      }
      if (bad_m | bad_v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (bad_m >> i & 1) mq[i] = __builtin_nanf("");
          if (bad_v >> i & 1) vq[i] = __builtin_nanf("");
        }
      }
      store_as<STREAM, uint32_t>((uint8_t *)p.m + base + at, pack_codes(mq));
      store_as<STREAM, uint32_t>((uint8_t *)p.v + base + at, pack_codes(vq));
      if (lane == 0) {
        p.m_scale[base / kTile + tile] = power_of_two(em);
        p.v_scale[base / kTile + tile] = power_of_two(ev);
      }
    } else {
      store_as<STREAM, f32x4>((float *)p.m + base + at, m);
      store_as<STREAM, f32x4>((float *)p.v + base + at, v);
    }
  }
}

template <typename W, typename G, bool EIGHT, int TILES, bool STREAM>
__global__ __launch_bounds__(kBlock) void adamw_kernel(AdamTable tab, AdamArgs p) {
  int lo = 0, hi = tab.count;                // the tensor of this workgroup
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const AdamSlice<W, G> s = {(W *)tab.w[lo], (const G *)tab.g[lo], tab.n[lo], tab.base[lo],
                             ((int64_t)(blockIdx.x - tab.first[lo]) * kWavesPerBlock + wave) * TILES, tab.keep[lo]};
  if (s.tile0 * kTile >= s.n) return;
  if ((s.tile0 + TILES) * kTile <= s.n) adamw_tiles<W, G, EIGHT, TILES, STREAM, true>(p, s);
  else adamw_tiles<W, G, EIGHT, TILES, STREAM, false>(p, s);
}

// The two terms of step t, t being counted on the device.
__global__ void adamw_terms_kernel(const uint64_t *t_dev, double lr, double b1, double b2, float *terms) {
  const double t = (double)*t_dev;
  terms[0] = (float)(lr / (1.0 - pow(b1, t)));
  terms[1] = (float)(1.0 / sqrt(1.0 - pow(b2, t)));
}

constexpr int64_t kAdamBlocks = (1ll << 32) / kBlock - 1;

// How much of the machine and of the caches a step takes.
enum Size { kSmall, kDeep, kStream };

template <typename W, typename G, bool EIGHT>
static void launch_adamw(Size size, unsigned blocks, const AdamTable &tab, const AdamArgs &p, hipStream_t stream) {
  if (size == kSmall) hipLaunchKernelGGL((adamw_kernel<W, G, EIGHT, 1, false>), dim3(blocks), dim3(kBlock), 0, stream, tab, p);
  else if (size == kDeep) hipLaunchKernelGGL((adamw_kernel<W, G, EIGHT, 4, false>), dim3(blocks), dim3(kBlock), 0, stream, tab, p);
  else hipLaunchKernelGGL((adamw_kernel<W, G, EIGHT, 4, true>), dim3(blocks), dim3(kBlock), 0, stream, tab, p);
}

template <typename W, typename G>
static void launch_adamw(bool eight, Size size, unsigned blocks, const AdamTable &tab, const AdamArgs &p, hipStream_t stream) {
  if (eight) launch_adamw<W, G, true>(size, blocks, tab, p, stream);
  else launch_adamw<W, G, false>(size, blocks, tab, p, stream);
}

template <typename W>
static void launch_adamw(int g, bool eight, Size size, unsigned blocks, const AdamTable &tab, const AdamArgs &p, hipStream_t stream) {
  if (g == GCNX_F32) launch_adamw<W, float>(eight, size, blocks, tab, p, stream);
  else if (g == GCNX_BF16) launch_adamw<W, __bf16>(eight, size, blocks, tab, p, stream);
  else launch_adamw<W, _Float16>(eight, size, blocks, tab, p, stream);
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
    // so that a tensor fits a launch on its own (launches hold fewer than 2^32 threads)
    GCNX_REQUIRE(x.n <= kAdamBlocks * kTile * kWavesPerBlock, GCNX_ERR_UNSUPPORTED, "adamw: tensor %lld is too large", (long long)i);
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
  // Tiles a wavefront has in flight: 4 where they fill the machine (8 wavefronts a
  // SIMD), else 1, so that more of it takes part.  A step over more than the 256 MiB
  // that the Infinity Cache holds (weights, gradients, state) streams past the caches:
  // nothing of it is there when the next step comes.  us streamed / not, fp32 with
  // 32-bit state: 362 M elements 1760 / 1890, 48 M 229 / 258, 24 M 118 / 129; still
  // 86 / 82 at 17 M (272 MB), and 75 / 69 at 14 M (224 MB), which does not stream; bf16
  // gradients and 8-bit state: 362 M 875 / 1010, 48 M 130 / 137, 24 M (192 MB) 70 / 68.
  const int64_t bytes = total * ((q->w_dtype == GCNX_F32 ? 4 : 2) + (q->g_dtype == GCNX_F32 ? 4 : 2) + (eight ? 2 : 8));
  const Size size = total / (4 * kTile) < 8 * 1024 ? kSmall : bytes <= (256ll << 20) ? kDeep : kStream;
  const int64_t per_block = (int64_t)kTile * kWavesPerBlock * (size == kSmall ? 1 : 4);
  for (int64_t i = 0; i < n_tensors;) {
    AdamTable tab = {};
    int64_t blocks = 0;
    for (; i < n_tensors && tab.count < kAdamTensors; ++i) {
      const gcnx_adamw_tensor &x = h_tensors[i];
      if (x.n == 0) continue;
      const int64_t more = ceil_div(x.n, per_block);
      if (blocks + more > kAdamBlocks) break;
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
    if (q->w_dtype == GCNX_F32) launch_adamw<float>(q->g_dtype, eight, size, (unsigned)blocks, tab, p, as_stream(stream));
    else if (q->w_dtype == GCNX_BF16) launch_adamw<__bf16>(q->g_dtype, eight, size, (unsigned)blocks, tab, p, as_stream(stream));
    else launch_adamw<_Float16>(q->g_dtype, eight, size, (unsigned)blocks, tab, p, as_stream(stream));
    GCNX_CHECK_LAUNCH();
  }
  return GCNX_OK;
}
