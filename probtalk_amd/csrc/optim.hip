// Optimizer over a list of tensors: the global gradient norm and one AdamW step, each a few launches whatever the number of
// tensors, with the two moments in 32 bits or in one byte a value.
//
//   norm = sqrt(sum over all tensors of g^2), coef = min(1, max_norm / (norm + 1e-6))
//   g' = coef g;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Both kernels stream: what bounds them is HBM (fp32: 4 bytes a value for the norm and 28 for the step, 16 with 8-bit moments).
// The list travels as kernel arguments (pointers, sizes and the first work unit of each tensor; AT tensors a launch, below the
// 4 KB that a launch is sure to take), so nothing is uploaded, nothing is kept between calls and a captured step owns its
// table.  A workgroup takes one unit of one tensor and finds the tensor by bisection over the scalar table.
// The step alone: 226 tensors of 40 M fp32 values 180 us, 6.2 TB/s (most gradients come from the Infinity Cache); with 8-bit moments 119 us,
// 5.4 TB/s; 310 tensors of 160 M bf16 values with 8-bit moments 370 us in a row, 4.3 TB/s (450 when traced launch by launch)
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "pt_common.h"

namespace pt {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// 8-bit moments.  A block of 256 values shares one fp32 scale = (largest magnitude) / TOP; a magnitude code is a float of four
// exponent bits and M mantissa bits over the quantum `scale`: code c < 2^M stands for c, else for (2^M + (c mod 2^M)) 2^(c / 2^M - 1).
// First moment: sign bit + M = 3 (TOP = 15 * 2^14).  Second moment, never negative: M = 4 (TOP = 31 * 2^14).
// The parameters and moments pass through the step once: streaming loads and stores keep the gradients, which the norm has just read,
// in the caches (norm and step over 40 M fp32 values: 281 -> 218 us, with 8-bit moments 266 -> 219 including the reading of them).
// Codes are rounded stochastically: with b2 = 0.999 a second moment moves by a thousandth per step, far less than half a code
// step (1/32 to 1/16 of the value), so rounding to nearest would leave it where it is for ever; a rounding whose MEAN is the
// value follows.  A positive second moment never becomes code 0 (its square root divides).  The 32 random bits of a value are a
// hash of (seed, step, position in the list), so a step is a function of its inputs.  All arithmetic that decides a code is
// plain IEEE fp32, one operation at a time (no contraction), so any implementation of these lines gives the same codes.
// ---------------------------------------------------------------------------
constexpr int QBLOCK = 256;
constexpr int M_BITS = 3, V_BITS = 4;
constexpr float TOP_M = 245760.f, TOP_V = 507904.f;
constexpr float SCALE_MIN = 7.888609052210118e-31f;   // 2^-100: a block whose largest magnitude is below is held as zeros

__device__ __forceinline__ unsigned hash_bits(unsigned c, unsigned key) {
  unsigned x = (c ^ key) * 0x9E3779B9u;
  x ^= x >> 15;
  x *= 0x6A09E667u;
  return x ^ (x >> 14);
}

template <int M>
__device__ __forceinline__ float code_value(unsigned c) {
  // with the code's exponent bits in the place of fp32's, fp32 reads the same number as a multiple of 2^-126-M, denormals included
  return ldexpf(__uint_as_float(c << (23 - M)), 126 + M);
}

// |x| -> code, z = |x| / scale in [0, TOP], r: 16 random bits
template <int M>
__device__ __forceinline__ unsigned value_code(float z, unsigned r) {
#pragma clang fp contract(off)
  const unsigned lin = (unsigned)(z + (float)r * 0x1p-16f);
  const unsigned flt = ((__float_as_uint(z) + (r << (7 - M))) >> (23 - M)) - ((126u + M) << M);
  return z < (float)(1 << M) ? lin : flt;
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp_umax(unsigned v) {
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true));
}
// the maximum over the wave in every lane, without the LDS crossbar
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
  v = dpp_umax<0xB1>(v);       // quad_perm [1,0,3,2]
  v = dpp_umax<0x4E>(v);       // quad_perm [2,3,0,1]
  v = dpp_umax<0x141>(v);      // row_half_mirror
  v = dpp_umax<0x140>(v);      // row_mirror
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(b[0], b[1]);
}

// ---------------------------------------------------------------------------
// The list
// ---------------------------------------------------------------------------
constexpr int AT = 60;                 // tensors per launch: 60 * 60 bytes of table
// Values per workgroup of the step: 4 waves x 2 blocks of 256, in registers that let 8 waves run on a SIMD (4 blocks, 5 waves: 40 M fp32 values
// 222.5 -> 218.3 us, 160 M bf16 with 8-bit moments 705 -> 697)
constexpr int UNIT = 2048;
constexpr int NORM_UNIT = 16384;       // values per workgroup of the norm

struct AdamTab {
  void* p[AT];
  const void* g[AT];
  void* m[AT];
  void* v[AT];
  float* s[AT];                        // 8-bit moments: scales [blocks][2] = first | second
  uint64_t n[AT];                      // values * 2 + (1 if every pointer allows the vector path)
  unsigned first[AT];                  // first unit of the tensor
  unsigned blk[AT];                    // first block of the tensor, counted over the whole list (random bits)
};
struct AdamHyper {
  int count;
  const float* gscale;                 // device scalar or null
  const float* dyn;                    // null, or {1 - b1^t, sqrt(1 - b2^t)} and the hash key on the device
  float lr, b1, b2, eps, wd, bc1, bc2_sqrt;
  unsigned key;
};
static_assert(sizeof(AdamTab) + sizeof(AdamHyper) <= 4096, "kernel arguments");

__host__ __device__ inline unsigned step_key(unsigned seed, unsigned step) {
  unsigned x = (step * 0x9E3779B9u) ^ seed;
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  return x ^ (x >> 15);
}

template <typename TAB>
__device__ __forceinline__ int find_tensor(const TAB& t, int count, unsigned unit) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= unit) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float bf2f(unsigned short x) { return __uint_as_float((unsigned)x << 16); }
// bf16 parameters are rounded stochastically too: the step of a parameter is mostly below half of its last bf16 bit
__device__ __forceinline__ unsigned short f2bf_sr(float x, unsigned r16) {
  const unsigned u = __float_as_uint(x);
  const unsigned odd = (u >> 16) | ((u & 0xFFFFu) ? 0x40u : 0u);                  // infinities stay, a NaN stays one
  return (unsigned short)((u & 0x7F800000u) == 0x7F800000u ? odd : (u + r16) >> 16);
}

// What a tensor without the vector path (odd address) or the last block of a tensor does: one value at a time
// NT: a streaming load
template <bool NT = false, typename T>
__device__ __forceinline__ void load4(const T* __restrict__ b, size_t e, size_t n, bool vec, float (&x)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 q = NT ? __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(b + e)) : *reinterpret_cast<const f32x4*>(b + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = q[i];
    } else {
      const u16x4 q = NT ? __builtin_nontemporal_load(reinterpret_cast<const u16x4*>(b + e)) : *reinterpret_cast<const u16x4*>(b + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = bf2f(q[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) x[i] = e + i < n ? b[e + i] : 0.f;
      else x[i] = e + i < n ? bf2f(b[e + i]) : 0.f;
    }
  }
}
__device__ __forceinline__ void store4(float* __restrict__ b, size_t e, size_t n, bool vec, const float (&x)[4]) {
  if (vec) {
    const f32x4 q = {x[0], x[1], x[2], x[3]};
    __builtin_nontemporal_store(q, reinterpret_cast<f32x4*>(b + e));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) if (e + i < n) b[e + i] = x[i];
  }
}
__device__ __forceinline__ void store4(unsigned short* __restrict__ b, size_t e, size_t n, bool vec, const unsigned short (&x)[4]) {
  if (vec) {
    const u16x4 q = {x[0], x[1], x[2], x[3]};
    __builtin_nontemporal_store(q, reinterpret_cast<u16x4*>(b + e));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) if (e + i < n) b[e + i] = x[i];
  }
}
__device__ __forceinline__ unsigned load4b(const unsigned char* __restrict__ b, size_t e, size_t n, bool vec) {
  if (vec) return __builtin_nontemporal_load(reinterpret_cast<const unsigned*>(b + e));
  unsigned x = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) if (e + i < n) x |= (unsigned)b[e + i] << (8 * i);
  return x;
}
__device__ __forceinline__ void store4b(unsigned char* __restrict__ b, size_t e, size_t n, bool vec, unsigned x) {
  if (vec) { __builtin_nontemporal_store(x, reinterpret_cast<unsigned*>(b + e)); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) if (e + i < n) b[e + i] = (unsigned char)(x >> (8 * i));
}

// the moments of the 8-bit form: one IEEE operation at a time
__device__ __forceinline__ void moments8(float g, float gs, float b1, float c1, float b2, float c2, float& m, float& v) {
#pragma clang fp contract(off)
  const float gr = g * gs;
  m = b1 * m + c1 * gr;
  v = b2 * v + (c2 * gr) * gr;
}

// the 32-bit form: every operation rounded by itself, the bits of adamw_kernel (train.hip)
__device__ __forceinline__ float adamw32(float p, float g, float gs, float b1, float c1, float b2, float c2, float decay, float step_size, float bc2_sqrt,
                                         float eps, float& m, float& v) {
#pragma clang fp contract(off)
  const float gr = g * gs;
  m = b1 * m + c1 * gr;
  v = b2 * v + c2 * gr * gr;
  const float denom = sqrtf(v) / bc2_sqrt + eps;
  return p * decay - step_size * (m / denom);
}

// One wave's 512 values of tensor i from e0 on.  T: float or bf16 bits (unsigned short); S8: 8-bit moments; FULL: all of them are there and
// aligned, so the loads are plain vectors and all of them go out before the first is waited for.
template <typename T, bool S8, bool FULL>
__device__ __forceinline__ void adamw_wave(const AdamTab& tab, const AdamHyper& h, const int i, const size_t e0, const size_t n) {
  const bool aligned = tab.n[i] & 1;
  const int lane = threadIdx.x & 63;
  T* __restrict__ P = (T*)tab.p[i];
  const T* __restrict__ G = (const T*)tab.g[i];
  const float gs = h.gscale ? *h.gscale : 1.f;
  float bc1 = h.bc1, bc2_sqrt = h.bc2_sqrt;
  unsigned key = h.key;
  if (h.dyn) { bc1 = h.dyn[0]; bc2_sqrt = h.dyn[1]; key = __float_as_uint(h.dyn[2]); }
  const float c1 = 1.f - h.b1, c2 = 1.f - h.b2;
  const float decay = fmaf(-h.lr, h.wd, 1.f), step_size = h.lr / bc1;
  constexpr int NB = UNIT / 4 / QBLOCK;                  // independent blocks of a wave: their loads are in flight together
  float p[NB][4], g[NB][4], m[NB][4], v[NB][4];
  unsigned cm[NB], cv[NB];
  float sm[NB], sv[NB];
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    const size_t e = e0 + k * QBLOCK + lane * 4;
    const bool vec = FULL || (aligned && e + 4 <= n);
    load4<true>(P, e, n, vec, p[k]);
    load4(G, e, n, vec, g[k]);
    if constexpr (S8) {
      cm[k] = load4b((const unsigned char*)tab.m[i], e, n, vec);
      cv[k] = load4b((const unsigned char*)tab.v[i], e, n, vec);
      const size_t b = e0 / QBLOCK + k;
      const bool in = FULL || b * QBLOCK < n;
      sm[k] = in ? tab.s[i][2 * b] : 0.f;
      sv[k] = in ? tab.s[i][2 * b + 1] : 0.f;
    } else {
      load4<true>((const float*)tab.m[i], e, n, vec, m[k]);
      load4<true>((const float*)tab.v[i], e, n, vec, v[k]);
    }
  }
  // 8-bit moments: the new moments of all blocks, then the scales of the (block, moment) pairs in as many lanes at once:
  // a division and a reciprocal cost ten instructions each, and every lane of the wave would compute the same
  float inv_m[NB], inv_v[NB];
  if constexpr (S8) {
    unsigned top[2 * NB];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      unsigned am = 0, av = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned c = cm[k] >> (8 * j);
        const float mag = code_value<M_BITS>(c & 127u) * sm[k];
        m[k][j] = c & 128u ? -mag : mag;
        v[k][j] = code_value<V_BITS>((cv[k] >> (8 * j)) & 255u) * sv[k];
        moments8(g[k][j], gs, h.b1, c1, h.b2, c2, m[k][j], v[k][j]);
        // as unsigned integers magnitudes order like the floats, and a NaN is the largest of all
        am = max(am, __float_as_uint(m[k][j]) & 0x7FFFFFFFu);
        av = max(av, __float_as_uint(v[k][j]) & 0x7FFFFFFFu);
      }
      top[2 * k] = wave_umax(am);
      top[2 * k + 1] = wave_umax(av);
    }
    unsigned mine = top[0];
#pragma unroll
    for (int i = 1; i < 2 * NB; ++i) mine = (lane & 7) == i ? top[i] : mine;
    const float big = __uint_as_float(mine);
    // a block with a NaN or an infinity: that scale, codes 0, NaN from here on
    const float scale = big < SCALE_MIN ? 0.f : big / (lane & 1 ? TOP_V : TOP_M);
    const float inv = big >= SCALE_MIN && big < INFINITY ? 1.f / scale : 0.f;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      sm[k] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scale), 2 * k));
      sv[k] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scale), 2 * k + 1));
      inv_m[k] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(inv), 2 * k));
      inv_v[k] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(inv), 2 * k + 1));
    }
  }
  const float bc2_inv = 1.f / bc2_sqrt;
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    const size_t e = e0 + k * QBLOCK + lane * 4;
    const bool vec = FULL || (aligned && e + 4 <= n);
    unsigned short pb[4];
    unsigned om = 0, ov = 0, sign = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float pv;
      if constexpr (S8) {
        // nothing here decides a code: the hardware's root and reciprocal (1 ulp each) for the IEEE ones' forty instructions
        const float denom = fmaf(__builtin_amdgcn_sqrtf(v[k][j]), bc2_inv, h.eps);
        pv = fmaf(decay, p[k][j], -(step_size * (m[k][j] * __builtin_amdgcn_rcpf(denom))));
      } else {
        pv = adamw32(p[k][j], g[k][j], gs, h.b1, c1, h.b2, c2, decay, step_size, bc2_sqrt, h.eps, m[k][j], v[k][j]);
      }
      p[k][j] = pv;
      unsigned r = 0;
      if constexpr (S8 || sizeof(T) == 2)
        r = hash_bits((tab.blk[i] + (unsigned)(e0 / QBLOCK) + k) * (unsigned)QBLOCK + lane * 4 + j, key);
      if constexpr (S8) {
        const float zm = fminf(fabsf(m[k][j]) * inv_m[k], TOP_M), zv = fminf(v[k][j] * inv_v[k], TOP_V);
        om |= value_code<M_BITS>(zm, r & 0xFFFFu) << (8 * j);
        ov |= max(value_code<V_BITS>(zv, r >> 16), zv > 0.f ? 1u : 0u) << (8 * j);
        sign |= (m[k][j] < 0.f ? 128u : 0u) << (8 * j);
      }
      if constexpr (sizeof(T) == 2) pb[j] = f2bf_sr(pv, ((r * 0xBB67AE85u) >> 16) & 0xFFFFu);
    }
    if constexpr (sizeof(T) == 2) store4((unsigned short*)P, e, n, vec, pb); else store4((float*)P, e, n, vec, p[k]);
    if constexpr (S8) {
      store4b((unsigned char*)tab.m[i], e, n, vec, (inv_m[k] > 0.f ? om : 0u) | sign);      // no finite scale: codes 0
      store4b((unsigned char*)tab.v[i], e, n, vec, inv_v[k] > 0.f ? ov : 0u);
      const size_t b = e0 / QBLOCK + k;
      if (lane == 0 && (FULL || b * QBLOCK < n)) { tab.s[i][2 * b] = sm[k]; tab.s[i][2 * b + 1] = sv[k]; }
    } else {
      store4((float*)tab.m[i], e, n, vec, m[k]);
      store4((float*)tab.v[i], e, n, vec, v[k]);
    }
  }
}

template <typename T, bool S8>
__global__ __launch_bounds__(256) void adamw_multi_kernel(const AdamTab tab, const AdamHyper h) {
  const int i = find_tensor(tab, h.count, blockIdx.x);
  const size_t n = (size_t)(tab.n[i] >> 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t e0 = (size_t)(blockIdx.x - tab.first[i]) * UNIT + wave * (UNIT / 4);
  if (e0 >= n) return;                                   // whole waves leave; nothing is shared between waves
  if ((tab.n[i] & 1) && e0 + UNIT / 4 <= n) adamw_wave<T, S8, true>(tab, h, i, e0, n);
  else adamw_wave<T, S8, false>(tab, h, i, e0, n);
}

// the step count of a captured step lives on the device
__global__ void adamw_dyn_kernel(const int* __restrict__ step, float b1, float b2, unsigned seed, float* __restrict__ dyn) {
  const int t = *step;
  dyn[0] = 1.f - (float)pow((double)b1, (double)t);
  dyn[1] = sqrtf(1.f - (float)pow((double)b2, (double)t));
  dyn[2] = __uint_as_float(step_key(seed, (unsigned)t));
}

int launch_adamw_multi(void* const* p, const void* const* g, void* const* m, void* const* v, float* const* scales, const int64_t* n,
                       int count, int dtype, const float* gscale, float lr, float beta1, float beta2, float eps, float wd, int step,
                       const int* step_dev, float* dyn, unsigned seed, hipStream_t s) {
  PT_CHECK(p && g && m && v && n && count >= 0 && (dtype == 0 || dtype == 1), "adamw_multi: bad argument");
  PT_CHECK(step_dev ? dyn != nullptr : step >= 1, "adamw_multi: step must be at least 1, and a step on the device needs its scratch");
  for (int i = 0; i < count; ++i)
    PT_CHECK(n[i] >= 0 && (n[i] == 0 || (p[i] && g[i] && m[i] && v[i] && (!scales || scales[i]))), "adamw_multi: null tensor %d", i);
  AdamHyper h = {};
  h.gscale = gscale;
  h.lr = lr; h.b1 = beta1; h.b2 = beta2; h.eps = eps; h.wd = wd;
  if (step_dev) {
    PT_LAUNCH(adamw_dyn_kernel, dim3(1), dim3(1), 0, s, step_dev, beta1, beta2, seed, dyn);
    h.dyn = dyn;
  } else {
    h.bc1 = 1.f - powf(beta1, (float)step);
    h.bc2_sqrt = sqrtf(1.f - powf(beta2, (float)step));
    h.key = step_key(seed, (unsigned)step);
  }
  const uintptr_t pmask = dtype ? 7 : 15, smask = scales ? 3 : 15;
  unsigned blk = 0;
  for (int i = 0; i < count;) {
    AdamTab t;
    unsigned units = 0;
    int k = 0;
    for (; i < count && k < AT; ++i) {
      if (n[i] == 0) continue;
      const uint64_t u = ((uint64_t)n[i] + UNIT - 1) / UNIT;
      PT_CHECK(u < (1u << 24), "adamw_multi: tensor %d has too many values", i);       // a launch holds less than 2^32 threads
      if (k && units + u >= (1u << 24)) break;
      t.p[k] = p[i]; t.g[k] = g[i]; t.m[k] = m[i]; t.v[k] = v[i]; t.s[k] = scales ? scales[i] : nullptr;
      const bool vec = !((((uintptr_t)p[i] | (uintptr_t)g[i]) & pmask) | (((uintptr_t)m[i] | (uintptr_t)v[i]) & smask));
      t.n[k] = (uint64_t)n[i] * 2 + (vec ? 1 : 0);
      t.first[k] = units;
      t.blk[k] = blk;
      units += (unsigned)u;
      blk += (unsigned)(((uint64_t)n[i] + QBLOCK - 1) / QBLOCK);
      ++k;
    }
    if (!k) break;
    h.count = k;
    if (scales) {
      if (dtype) PT_LAUNCH((adamw_multi_kernel<unsigned short, true>), dim3(units), dim3(256), 0, s, t, h);
      else PT_LAUNCH((adamw_multi_kernel<float, true>), dim3(units), dim3(256), 0, s, t, h);
    } else {
      if (dtype) PT_LAUNCH((adamw_multi_kernel<unsigned short, false>), dim3(units), dim3(256), 0, s, t, h);
      else PT_LAUNCH((adamw_multi_kernel<float, false>), dim3(units), dim3(256), 0, s, t, h);
    }
  }
  return 0;
}

// ---------------------------------------------------------------------------
// What 8-bit moments stand for, as fp32 (checkpoints, inspection): one thread per four values
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void moment_values_kernel(const unsigned char* __restrict__ m, const unsigned char* __restrict__ v,
                                                            const float* __restrict__ s, size_t n, int vec, float* __restrict__ mo,
                                                            float* __restrict__ vo) {
  const size_t e = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= n) return;
  const bool w = vec && e + 4 <= n;
  const unsigned a = load4b(m, e, n, w), b = load4b(v, e, n, w);
  const float sm = s[2 * (e / QBLOCK)], sv = s[2 * (e / QBLOCK) + 1];
  float x[4], y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned c = (a >> (8 * j)) & 255u;
    const float mag = code_value<M_BITS>(c & 127u) * sm;
    x[j] = c & 128u ? -mag : mag;
    y[j] = code_value<V_BITS>((b >> (8 * j)) & 255u) * sv;
  }
  store4(mo, e, n, w, x);
  store4(vo, e, n, w, y);
}
int launch_moment_values(const unsigned char* m, const unsigned char* v, const float* scales, int64_t n, float* m_out, float* v_out,
                         hipStream_t s) {
  PT_CHECK(n >= 0 && n < ((int64_t)1 << 34) && (n == 0 || (m && v && scales && m_out && v_out)), "moment_values: bad argument");
  if (n == 0) return 0;
  const int vec = !(((uintptr_t)m | (uintptr_t)v) & 3) && !(((uintptr_t)m_out | (uintptr_t)v_out) & 15);
  PT_LAUNCH(moment_values_kernel, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, s, m, v, scales, (size_t)n, vec, m_out, v_out);
  return 0;
}

// ---------------------------------------------------------------------------
// Global gradient norm.  Squares are exact in fp64 and summed there (fp64 runs at the fp32 rate on this chip's vector unit and
// the kernel is bound by HBM), one partial sum per workgroup in the caller's scratch; one workgroup adds the partials in a fixed
// order, so the same gradients give the same bits.
// ---------------------------------------------------------------------------
constexpr int NT = 180;                // tensors per launch: 180 * 20 bytes of table
struct NormTab {
  const void* g[NT];
  uint64_t n[NT];                      // values * 4 + 2 if bf16 + 1 if aligned
  unsigned first[NT];
};
static_assert(sizeof(NormTab) + 32 <= 4096, "kernel arguments");

__device__ __forceinline__ double wave_dsum(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ double sumsq_unit(const T* __restrict__ g, size_t e0, size_t n, bool aligned, int thread) {
  double s[4] = {0, 0, 0, 0};
  const size_t end = min(n, e0 + (size_t)NORM_UNIT);
  if (aligned && end == e0 + NORM_UNIT) {
    g += e0 + thread * 4;
#pragma unroll 8
    for (int k = 0; k < NORM_UNIT / 1024; ++k) {
      float x[4];
      load4(g, (size_t)k * 1024, 0, true, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = fma((double)x[j], (double)x[j], s[j]);
    }
  } else {
    for (size_t e = e0 + thread * 4; e < end; e += 1024) {
      float x[4];
      load4(g, e, n, aligned && e + 4 <= n, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = fma((double)x[j], (double)x[j], s[j]);
    }
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ __forceinline__ double sumsq_unit(const NormTab& tab, int count, unsigned unit, int thread) {
  const int i = find_tensor(tab, count, unit);
  const size_t n = (size_t)(tab.n[i] >> 2), e0 = (size_t)(unit - tab.first[i]) * NORM_UNIT;
  const bool aligned = tab.n[i] & 1;
  return tab.n[i] & 2 ? sumsq_unit((const unsigned short*)tab.g[i], e0, n, aligned, thread) : sumsq_unit((const float*)tab.g[i], e0, n, aligned, thread);
}
__global__ __launch_bounds__(256) void grad_sumsq_kernel(const NormTab tab, int count, double* __restrict__ part) {
  const double s = wave_dsum(sumsq_unit(tab, count, blockIdx.x, threadIdx.x));
  __shared__ double red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}
// norm and coefficient from the sums of a workgroup of 1024 threads
__device__ __forceinline__ void norm_out(double s, float max_norm, float* __restrict__ norm, float* __restrict__ coef) {
  s = wave_dsum(s);
  __shared__ double red[16];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) s += red[w];
    const float nrm = (float)sqrt(s);
    const float c = max_norm / (nrm + 1e-6f);
    *norm = nrm;
    *coef = c > 1.f ? 1.f : c;                           // a norm that is no number gives a coefficient that is none
  }
}
__global__ __launch_bounds__(1024) void grad_norm_kernel(const double* __restrict__ part, unsigned units, float max_norm,
                                                         float* __restrict__ norm, float* __restrict__ coef) {
  double s = 0;
  for (unsigned u = threadIdx.x; u < units; u += 1024) s += part[u];
  norm_out(s, max_norm, norm, coef);
}
// A few units (a head, an adapter): one workgroup, four units at a time, and no second launch: 3 units 4.97 -> 3.93 us, 8 units 5.1 -> 6.3, but one
// launch of some 4 us less for the host, which is the bound of such calls (3 units with their step: 21.8 -> 18.6 us a call)
constexpr unsigned FEW_UNITS = 8;
__global__ __launch_bounds__(1024) void grad_norm_few_kernel(const NormTab tab, int count, unsigned units, float max_norm, float* __restrict__ norm,
                                                             float* __restrict__ coef) {
  double s = 0;
  for (unsigned u = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8); u < units; u += 4) s += sumsq_unit(tab, count, u, threadIdx.x & 255);
  norm_out(s, max_norm, norm, coef);
}

static uint64_t norm_units(int64_t n) { return ((uint64_t)n + NORM_UNIT - 1) / NORM_UNIT; }

size_t grad_norm_workspace(const int64_t* n, int count) {
  uint64_t u = 0;
  for (int i = 0; i < count; ++i) u += n[i] > 0 ? norm_units(n[i]) : 0;
  return (size_t)(u ? u : 1) * sizeof(double);
}

int launch_grad_norm(const void* const* g, const int64_t* n, const unsigned char* is_bf16, int count, float max_norm, float* norm,
                     float* coef, void* ws, size_t ws_bytes, hipStream_t s) {
  PT_CHECK(count >= 0 && (count == 0 || (g && n)) && norm && coef && ws, "grad_norm: bad argument");
  for (int i = 0; i < count; ++i) PT_CHECK(n[i] >= 0 && (n[i] == 0 || g[i]), "grad_norm: null tensor %d", i);
  PT_CHECK(ws_bytes >= grad_norm_workspace(n, count) && ((uintptr_t)ws & 7) == 0, "grad_norm: workspace of %zu bytes, %zu needed",
           ws_bytes, grad_norm_workspace(n, count));
  PT_CHECK(grad_norm_workspace(n, count) / sizeof(double) < (1u << 31), "grad_norm: too many values");
  double* part = (double*)ws;
  unsigned done = 0;
  for (int i = 0; i < count;) {
    NormTab t;
    unsigned units = 0;
    int k = 0;
    for (; i < count && k < NT; ++i) {
      if (n[i] == 0) continue;
      const bool b = is_bf16 && is_bf16[i];
      t.g[k] = g[i];
      t.n[k] = (uint64_t)n[i] * 4 + (b ? 2 : 0) + (((uintptr_t)g[i] & (b ? 7 : 15)) ? 0 : 1);
      t.first[k] = units;
      units += (unsigned)norm_units(n[i]);
      ++k;
    }
    if (!k) break;
    if (done == 0 && i == count && units <= FEW_UNITS) {
      PT_LAUNCH(grad_norm_few_kernel, dim3(1), dim3(1024), 0, s, t, k, units, max_norm, norm, coef);
      return 0;
    }
    PT_LAUNCH(grad_sumsq_kernel, dim3(units), dim3(256), 0, s, t, k, part + done);
    done += units;
  }
  PT_LAUNCH(grad_norm_kernel, dim3(1), dim3(1024), 0, s, part, done, max_norm, norm, coef);
  return 0;
}

}  // namespace pt
