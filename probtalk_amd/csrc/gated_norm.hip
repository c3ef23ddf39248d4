// Norm of a block's output, gate, residual scale, residual sum and the norm in front of the next block, in one pass:
//
//   u = N(t) w1 + b1,   y = x + a g u,   h = N(y) w2 + b2          N: LayerNorm or RMSNorm over the row
//
// with one gate row g per clip (rows_per_clip rows share it) and one residual scale a per column.  Left out parts: t (y = x), g, a
// (ones), w1 (u = t), w2 (no h).  Backward, with dn = dh w2 and "bar" the mean over the row (its first term only for LayerNorm):
//
//   D  = dy + r_y (dn - bar(dn) - y^ bar(dn y^))                    dx = D
//   dm = D a g w1,  dt = r_t (dm - bar(dm) - t^ bar(dm t^))
//   dw2 = sum dh y^, db2 = sum dh, dw1 = a sum g D t^, db1 = a sum g D, da = w1 sum g D t^ + b1 sum g D, dg = sum over the clip of D a u
//
// Bound by HBM: forward 2 rows in and 2 out, backward 4 in and 2 out.  y and the statistics' arguments are recomputed from x and t
// (the same bytes as reading a stored y, and exact where y is held in bf16); only 4 floats a row are kept from the forward pass.
//
// A row is held by L lanes (8 to 512), PER values each; a worker (these lanes) walks a run of rows, so the column vectors stay in registers
// and the column sums of the backward pass are register adds.  A worker's rows lie in one clip, or are whole clips, so the gate's
// gradient is a register sum too, stored once per clip (or joined within the block, and added up in order by the second kernel with
// the other column sums).  No atomics: the same inputs give the same bits.
//
// Measured: 49,152 x 2048 bf16 forward 180 us (4.5 TB/s; a copy of this size runs at 4.9); 45,056 x 512 fp32 forward 80 us (4.6 TB/s;
// 64 where its inputs lie in the caches), with all gradients 195; 16,384 x 4096 bf16 with gradients 290; lanes to the row's length:
// 200,000 x 64 bf16 forward 107 -> 27 us, with gradients 349 -> 189
#include <algorithm>
#include <cstdint>

#include "pt_common.h"

namespace pt {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

struct GatedArgs {
  const void* x; const void* t; const void* gate;
  const float* a; const float* w1; const float* b1; const float* w2; const float* b2;
  const void* dy; const void* dh;
  void* y; void* h; float* stats;      // stats [rows][4]: mean t, 1/std t, mean y, 1/std y
  void* dx; void* dt; void* dgate;
  float* part;                         // [blocks][4][cols]: sum g D t^ | sum g D | sum dh y^ | sum dh
  float* gpart;                        // [workers][cols] (joined: [blocks][cols]): shares of a clip's gate gradient, or null (whole clips)
  size_t ldx, ldt;
  int rows, cols, clip;                // rows per clip (of the gate)
  int run, spc;                        // rows per worker; workers per clip, or 0: a worker takes run / clip whole clips
  int joined;                          // a block's workers are all of one clip: they share one row of gpart
  float eps;
  int layer;                           // LayerNorm, else RMSNorm
  int stream;                          // see store_row
};

template <int CTRL>
__device__ __forceinline__ float dpp_sum(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// sum over L lanes (64: the wave), the same in every one, without the LDS crossbar
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  v = dpp_sum<0xB1>(v);        // quad_perm [1,0,3,2]
  v = dpp_sum<0x4E>(v);        // quad_perm [2,3,0,1]
  v = dpp_sum<0x141>(v);       // row_half_mirror
  if constexpr (L >= 16) v = dpp_sum<0x140>(v);        // row_mirror
  if constexpr (L == 32) {
    const unsigned u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned a0 = a[0], a1 = a[1];
    v = __uint_as_float(a0) + __uint_as_float(a1);
  }
  if constexpr (L >= 64) v = row_lanes_sum(v);
  return v;
}

template <int L>
struct RowSum {
  static constexpr int WPR = L / 64;    // waves of a row
  float* slot;                         // LDS [2][RPB][WPR][2]
  int flip = 0;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    a = lanes_sum<L>(a);
    b = lanes_sum<L>(b);
    if constexpr (WPR > 1) {
      // two slots in turn: a slot is written again only behind the barrier of the other one, which every reader has passed
      float* s = slot + flip * 2 * (blockDim.x >> 6);
      flip ^= 1;
      const int wave = threadIdx.x >> 6, first = wave / WPR * WPR;
      if ((threadIdx.x & 63) == 0) { s[2 * wave] = a; s[2 * wave + 1] = b; }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) { a += s[2 * (first + w)]; b += s[2 * (first + w) + 1]; }
    }
  }
};

// columns of a lane: chunks of 16 bytes, neighbouring lanes next to each other
template <typename T, int L, int PER>
__device__ __forceinline__ int column(int i) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x % L;
  return (i / V * L + lane) * V + i % V;
}

__device__ __forceinline__ unsigned short to_bf16(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }

// How rows are read and written: 16 bytes at a time from 16-byte addresses, 16 bytes from any (columns or strides that are no multiples of 16
// bytes; the hardware takes them), or value by value (rows of less than 16 bytes)
enum Access { ALIGNED, ANY, SCALAR };
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <typename T> struct Chunk;
template <> struct Chunk<float> { typedef u32x4 any __attribute__((aligned(4))); static constexpr int V = 4; };
template <> struct Chunk<unsigned short> { typedef u32x4 any __attribute__((aligned(2))); static constexpr int V = 8; };

// a lane's values of a row as they lie in memory: what is loaded ahead waits in half the registers where it is bf16
template <typename T, int L, int PER, int ACC>
struct Raw {
  static constexpr int V = Chunk<T>::V, N = PER / V;
  u32x4 x[N];
  __device__ __forceinline__ void load(const T* __restrict__ p, int cols) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int c0 = column<T, L, PER>(c * V);
      // lanes behind the last column read the last ones again: nothing they compute is summed up or stored, and a load without
      // a branch is one that nobody waits for before its value is needed
      if constexpr (ACC == ALIGNED) x[c] = *reinterpret_cast<const u32x4*>(p + min(c0, cols - V));
      else if constexpr (ACC == ANY) x[c] = *reinterpret_cast<const typename Chunk<T>::any*>(p + min(c0, cols - V));
      else {
        x[c] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c0 + j < cols) {
            if constexpr (V == 4) x[c][j] = __float_as_uint(p[c0 + j]);
            else x[c][j / 2] |= (unsigned)p[c0 + j] << (16 * (j & 1));
          }
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[PER], int cols) const {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      u32x4 y = x[c];
      if constexpr (ACC == ANY) {
        // the lane across the row's end read from cols - V on: down by what that is too early
        const int early = column<T, L, PER>(c * V) + V - cols, by = early > 0 && early < V ? early : 0;
        if constexpr (V == 8) {
          const u32x4 s = {y[0] >> 16 | y[1] << 16, y[1] >> 16 | y[2] << 16, y[2] >> 16 | y[3] << 16, y[3] >> 16};
          y = by & 1 ? s : y;
        }
        y = by & V / 4 ? u32x4{y[1], y[2], y[3], y[3]} : y;
        y = by & V / 2 ? u32x4{y[2], y[3], y[3], y[3]} : y;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if constexpr (V == 4) { const unsigned u = y[j]; v[c * V + j] = __uint_as_float(u); }
        else { const unsigned u = y[j / 2]; v[c * V + j] = __uint_as_float(j & 1 ? u & 0xFFFF0000u : u << 16); }
      }
    }
  }
};
template <typename T, int L, int PER, int ACC>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int cols, float (&v)[PER]) {
  Raw<T, L, PER, ACC> r;
  r.load(p, cols);
  r.get(v, cols);
}
template <typename Q>
__device__ __forceinline__ void put(Q* p, const Q& q, bool stream) {
  if (stream) {
    asm volatile("");                  // the compiler makes one plain store of the two otherwise
    __builtin_nontemporal_store(q, p);
    asm volatile("");
  } else {
    *p = q;
  }
}
// stream: outputs larger than the caches, which would only push out what is read again
template <typename T, int L, int PER, int ACC>
__device__ __forceinline__ void store_row(T* __restrict__ p, int cols, const float (&v)[PER], bool stream = false) {
  constexpr int V = Chunk<T>::V;
#pragma unroll
  for (int c = 0; c < PER / V; ++c) {
    const int c0 = column<T, L, PER>(c * V);
    unsigned short b[V];
    if constexpr (V == 8)
#pragma unroll
      for (int j = 0; j < V; ++j) b[j] = to_bf16(v[c * V + j]);
    if (ACC != SCALAR && c0 + V <= cols) {
      u32x4 q;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (V == 4) q[j] = __float_as_uint(v[c * V + j]);
        else q[j] = b[2 * j] | (unsigned)b[2 * j + 1] << 16;
      }
      if constexpr (ACC == ALIGNED) put(reinterpret_cast<u32x4*>(p + c0), q, stream);
      else *reinterpret_cast<typename Chunk<T>::any*>(p + c0) = q;
    } else if (ACC != ALIGNED) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c0 + j < cols) {
          if constexpr (V == 4) p[c0 + j] = v[c * V + j];
          else p[c0 + j] = b[j];
        }
    }
  }
}
// a column vector in fp32 at the columns of T's chunks; `fill` where there is none
template <typename T, int L, int PER>
__device__ __forceinline__ void load_cols(const float* __restrict__ p, int cols, float fill, float (&v)[PER]) {
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = column<T, L, PER>(i);
    v[i] = p ? (c < cols ? p[c] : 0.f) : fill;
  }
}

// rows [r0, r1) of a worker; workers behind the last one get none
__device__ __forceinline__ void worker_rows(const GatedArgs& g, int worker, int& r0, int& r1) {
  int64_t begin = (int64_t)worker * g.run, end = begin + g.run, most = g.rows;
  if (g.spc) {
    const int clip = worker / g.spc, seg = worker - clip * g.spc;
    begin = (int64_t)clip * g.clip + (int64_t)seg * g.run;
    end = begin + g.run;
    most = min(most, ((int64_t)clip + 1) * g.clip);
  }
  r0 = (int)min(begin, most);
  r1 = (int)min(end, most);
}

// mean and 1/std of the values; what lies behind the last column is kept out of the sums
template <typename T, int L, int PER, bool LAYER>
__device__ __forceinline__ void row_stats(const float (&v)[PER], int cols, float inv_cols, float eps, RowSum<L>& sum, float& mean, float& rstd) {
  mean = 0.f;
  if constexpr (LAYER) {
    float s = 0.f, z = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) s += column<T, L, PER>(i) < cols ? v[i] : 0.f;
    sum(s, z);
    mean = s * inv_cols;
  }
  float q = 0.f, z = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float d = column<T, L, PER>(i) < cols ? v[i] - mean : 0.f;
    q += d * d;
  }
  sum(q, z);
  rstd = 1.f / sqrtf(q * inv_cols + eps);
}

template <typename T, int L, int PER, bool LAYER, int ACC>
__global__ __launch_bounds__(L > 256 ? L : 256) void gated_norm_fwd_kernel(const GatedArgs g) {
  constexpr int THREADS = L > 256 ? L : 256, RPB = THREADS / L;
  __shared__ float red[2 * 2 * (THREADS / 64)];
  RowSum<L> sum{red};
  int r0, r1;
  worker_rows(g, blockIdx.x * RPB + threadIdx.x / L, r0, r1);
  const int cols = g.cols;
  const float inv_cols = 1.f / (float)cols;
  const T* __restrict__ X = (const T*)g.x;
  const T* __restrict__ Tt = (const T*)g.t;
  float a[PER], w1[PER], b1[PER], w2[PER], b2[PER], gt[PER];
  load_cols<T, L, PER>(g.a, cols, 1.f, a);
  load_cols<T, L, PER>(g.w1, cols, 1.f, w1);
  load_cols<T, L, PER>(g.b1, cols, 0.f, b1);
  load_cols<T, L, PER>(g.w2, cols, 1.f, w2);
  load_cols<T, L, PER>(g.b2, cols, 0.f, b2);
#pragma unroll
  for (int i = 0; i < PER; ++i) gt[i] = a[i];
  Raw<T, L, PER, ACC> nx, nt;                               // without t: x in its place, not used
  auto fetch = [&](unsigned row) {
    row = min(row, (unsigned)g.rows - 1u);
    nx.load(X + (size_t)row * g.ldx, cols);
    nt.load(Tt ? Tt + (size_t)row * g.ldt : X + (size_t)row * g.ldx, cols);
  };
  fetch(r0);
  int left = 0;                                          // rows left of the current clip
  for (int k = 0; k < g.run; ++k) {                      // the same count for every worker of the block: barriers inside
    const unsigned row = (unsigned)r0 + k;               // behind the worker's last row it may pass 2^31
    const bool on = k < r1 - r0;
    float x[PER], t[PER];
    nx.get(x, cols);
    nt.get(t, cols);
    fetch(row + 1);
    if (g.gate && on && left == 0) {
      const int clip = (int)row / g.clip;
      left = (clip + 1) * g.clip - (int)row;
      load_row<T, L, PER, ACC>((const T*)g.gate + (size_t)clip * cols, cols, gt);
#pragma unroll
      for (int i = 0; i < PER; ++i) gt[i] *= a[i];
    }
    --left;
    if (!on) {
#pragma unroll
      for (int i = 0; i < PER; ++i) { x[i] = 0.f; t[i] = 0.f; }
    }
    float mt = 0.f, rt = 1.f, my = 0.f, ry = 1.f;
    if (Tt) {
      if (g.w1) {
        row_stats<T, L, PER, LAYER>(t, cols, inv_cols, g.eps, sum, mt, rt);
#pragma unroll
        for (int i = 0; i < PER; ++i) t[i] = (t[i] - mt) * rt * w1[i] + b1[i];
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] += gt[i] * t[i];
      if (on) store_row<T, L, PER, ACC>((T*)g.y + (size_t)row * cols, cols, x, g.stream);
    }
    if (g.w2) {
      // from the sum in fp32, not from the stored y: one rounding less in h
      row_stats<T, L, PER, LAYER>(x, cols, inv_cols, g.eps, sum, my, ry);
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = (x[i] - my) * ry * w2[i] + b2[i];
      if (on) store_row<T, L, PER, ACC>((T*)g.h + (size_t)row * cols, cols, x, g.stream);
    }
    if (g.stats && on && threadIdx.x % L == 0) {
      const f32x4 s = {mt, rt, my, ry};
      *reinterpret_cast<f32x4*>(g.stats + (size_t)row * 4) = s;
    }
  }
}

// BIAS: with biases (b1, or a bias' gradient is wanted)
template <typename T, int L, int PER, int ACC, bool BIAS>
__global__ __launch_bounds__(L > 256 ? L : 256, 2) void gated_norm_bwd_kernel(const GatedArgs g) {
  constexpr int THREADS = L > 256 ? L : 256, RPB = THREADS / L;
  __shared__ float red[2 * 2 * (THREADS / 64)];
  __shared__ float join[RPB > 1 ? RPB * L * PER : 1];
  RowSum<L> sum{red};
  const int worker = blockIdx.x * RPB + threadIdx.x / L;
  int r0, r1;
  worker_rows(g, worker, r0, r1);
  const int cols = g.cols;
  const float inv_cols = 1.f / (float)cols;
  const T* __restrict__ X = (const T*)g.x;
  const T* __restrict__ Tt = (const T*)g.t;
  const T* __restrict__ DY = (const T*)g.dy;
  const T* __restrict__ DH = (const T*)g.dh;
  // 16 values a lane: with the column vectors in registers too the kernel would spill, so these lie in LDS, where every lane reads what
  // it put there itself; and where the next row's loads do not fit either, they do not run ahead
  constexpr bool WIDE = PER > 8, AHEAD = !WIDE || (sizeof(T) == 2 && !BIAS);
  extern __shared__ __attribute__((aligned(16))) float wide[];           // [4][PER / 4][L][4]: w1 a, w2, gate, b1 a
  float w1[PER], b1[PER], w2[PER], gt[PER];              // w1 a, b1 a, w2, the gate
  {
    float a[PER];
    load_cols<T, L, PER>(g.a, cols, 1.f, a);
    load_cols<T, L, PER>(g.w1, cols, 1.f, w1);
    if constexpr (BIAS) load_cols<T, L, PER>(g.b1, cols, 0.f, b1);
    load_cols<T, L, PER>(g.w2, cols, 1.f, w2);
#pragma unroll
    for (int i = 0; i < PER; ++i) { w1[i] *= a[i]; b1[i] = BIAS ? b1[i] * a[i] : 0.f; }
  }
  auto wide_at = [&](int q, int i) { return wide + ((q * (PER / 4) + i / 4) * L + threadIdx.x % L) * 4 + i % 4; };
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      *wide_at(0, i) = w1[i];
      *wide_at(1, i) = w2[i];
      *wide_at(2, i) = 1.f;
      if constexpr (BIAS) *wide_at(3, i) = b1[i];
    }
  }
  // a column vector for the next use, from where it is held
  auto again = [&](int q, float (&v)[PER]) {
    if constexpr (WIDE) {
      asm volatile("" ::: "memory");                       // a read of its own, not one kept in registers
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = *wide_at(q, i);
    }
  };
  float aw[PER], ab[PER], bw[PER], bb[PER], dg[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) { gt[i] = 1.f; aw[i] = ab[i] = bw[i] = bb[i] = dg[i] = 0.f; }
  Raw<T, L, PER, ACC> nx, nt, ny, nh;
  f32x4 ns = {0.f, 0.f, 0.f, 0.f};
  auto fetch = [&](unsigned row) {                       // what is left out: x in its place, not used
    row = min(row, (unsigned)g.rows - 1u);
    const T* x = X + (size_t)row * g.ldx;
    nx.load(x, cols);
    nt.load(Tt ? Tt + (size_t)row * g.ldt : x, cols);
    ny.load(DY ? DY + (size_t)row * cols : x, cols);
    nh.load(DH ? DH + (size_t)row * cols : x, cols);
    ns = *reinterpret_cast<const f32x4*>(g.stats + (size_t)row * 4);
  };
  if (AHEAD) fetch(r0);
  int left = 0, clip = 0;
  for (int k = 0; k < g.run; ++k) {
    const unsigned row = (unsigned)r0 + k;               // behind the worker's last row it may pass 2^31
    const bool on = k < r1 - r0;
    if (!AHEAD) fetch(row);
    float x[PER], t[PER], dy[PER], dh[PER];
    const f32x4 st = on ? ns : f32x4{0.f, 0.f, 0.f, 0.f};   // another's row: its statistics may be no numbers, and 0 times these none either
    nx.get(x, cols);
    nt.get(t, cols);
    ny.get(dy, cols);
    nh.get(dh, cols);
    if (!on || !DY)
#pragma unroll
      for (int i = 0; i < PER; ++i) dy[i] = 0.f;
    if (!on || !Tt)
#pragma unroll
      for (int i = 0; i < PER; ++i) t[i] = 0.f;
    if (!on)                                               // a row that is another's: finite or not, it adds nothing
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = dh[i] = 0.f;
    if (AHEAD) fetch(row + 1);
    if (g.gate && on && left == 0) {
      clip = (int)row / g.clip;
      left = (clip + 1) * g.clip - (int)row;
      load_row<T, L, PER, ACC>((const T*)g.gate + (size_t)clip * cols, cols, gt);
      if constexpr (WIDE)
#pragma unroll
        for (int i = 0; i < PER; ++i) *wide_at(2, i) = gt[i];
    }
    --left;
    again(0, w1);
    again(2, gt);
    if constexpr (BIAS) again(3, b1);
    again(1, w2);
    // t: t^, x: y^
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      t[i] = g.w1 ? (t[i] - st[0]) * st[1] : t[i];
      x[i] += gt[i] * (t[i] * w1[i] + (BIAS ? b1[i] : 0.f));
      x[i] = (x[i] - st[2]) * st[3];
      const float dn = column<T, L, PER>(i) < cols ? dh[i] * w2[i] : 0.f;
      s1 += dn;
      s2 += dn * x[i];
    }
    if (DH) {
      sum(s1, s2);
      again(1, w2);
      const float m1 = g.layer ? s1 * inv_cols : 0.f, m2 = s2 * inv_cols;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        bw[i] += dh[i] * x[i];
        if constexpr (BIAS) bb[i] += dh[i];
        dy[i] += st[3] * (dh[i] * w2[i] - m1 - x[i] * m2);
      }
    }
    if (on) store_row<T, L, PER, ACC>((T*)g.dx + (size_t)row * cols, cols, dy, g.stream);
    if (Tt) {
      float s3 = 0.f, s4 = 0.f;
      again(0, w1);
      again(2, gt);
      if constexpr (BIAS) again(3, b1);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const float d = on && column<T, L, PER>(i) < cols ? dy[i] : 0.f, gd = gt[i] * d;
        aw[i] += gd * t[i];
        if constexpr (BIAS) ab[i] += gd;
        dg[i] += d * (t[i] * w1[i] + (BIAS ? b1[i] : 0.f));
        dy[i] = gd * w1[i];                              // the gradient of t^
        s3 += dy[i];
        s4 += dy[i] * t[i];
      }
      if (g.w1) {
        sum(s3, s4);
        const float m3 = g.layer ? s3 * inv_cols : 0.f, m4 = s4 * inv_cols;
#pragma unroll
        for (int i = 0; i < PER; ++i) dy[i] = st[1] * (dy[i] - m3 - t[i] * m4);
      }
      if (on && g.dt) store_row<T, L, PER, ACC>((T*)g.dt + (size_t)row * cols, cols, dy, g.stream);
    }
    if (g.dgate && on && !g.joined && (left == 0 || k + 1 == r1 - r0)) {
      if (g.gpart) {
#pragma unroll
        for (int i = 0; i < PER; ++i) if (column<T, L, PER>(i) < cols) g.gpart[(size_t)worker * cols + column<T, L, PER>(i)] = dg[i];
      } else {
        store_row<T, L, PER, ACC>((T*)g.dgate + (size_t)clip * cols, cols, dg);
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) dg[i] = 0.f;
    }
  }
  // this block's column sums
  float* __restrict__ out = g.part + (size_t)blockIdx.x * 4 * cols;
#pragma unroll
  for (int q = 0; q < 5; ++q) {
    if ((!BIAS && (q == 1 || q == 3)) || (q == 4 && !g.joined)) continue;
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = q == 0 ? aw[i] : q == 1 ? ab[i] : q == 2 ? bw[i] : q == 3 ? bb[i] : dg[i];
    float* to = q < 4 ? out + (size_t)q * cols : g.gpart + (size_t)blockIdx.x * cols;
    if constexpr (RPB > 1) {
      const int lane = threadIdx.x % L, who = threadIdx.x / L;
      __syncthreads();
      if (who)
#pragma unroll
        for (int i = 0; i < PER; ++i) join[(who * PER + i) * L + lane] = v[i];
      __syncthreads();
      if (!who)
#pragma unroll 3
        for (int w = 1; w < RPB; ++w)
#pragma unroll
          for (int i = 0; i < PER; ++i) v[i] += join[(w * PER + i) * L + lane];
      if (who) continue;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) if (column<T, L, PER>(i) < cols) to[column<T, L, PER>(i)] = v[i];
  }
}

// Adds the blocks' column sums (grid part 1: 64 columns and one of the two norms per block, 16 waves share the blocks) and the
// shares of each clip's gate gradient (part 2: 1024 columns of one clip per block, or from 32 shares on 64 columns and 16 waves that
// share them out).
constexpr int GATE_MANY = 32;
struct GatedFinish {
  const float* part; const float* gpart;
  const float* a; const float* w1; const float* b1;
  float* da; float* dw1; float* db1; float* dw2; float* db2;
  void* dgate;
  int blocks, cols, spc;
  int col_blocks, n_first;             // part 1: 2 * col_blocks blocks
};
template <typename T>
__global__ __launch_bounds__(1024) void gated_norm_finish_kernel(const GatedFinish f) {
  if ((int)blockIdx.x < f.n_first) {
    const int which = blockIdx.x / f.col_blocks, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = (blockIdx.x - which * f.col_blocks) * 64 + lane;
    float p = 0.f, q = 0.f;
    if (c < f.cols) {
      const float* s = f.part + (size_t)which * 2 * f.cols + c;
#pragma unroll 8
      for (int b = wave; b < f.blocks; b += 16) {
        p += s[(size_t)b * 4 * f.cols];
        q += s[(size_t)b * 4 * f.cols + f.cols];             // not written without biases, and then not used
      }
    }
    __shared__ float red[2][16][64];
    red[0][wave][lane] = p;
    red[1][wave][lane] = q;
    __syncthreads();
    if (wave || c >= f.cols) return;
    p = q = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) { p += red[0][w][lane]; q += red[1][w][lane]; }
    if (which) {
      if (f.dw2) f.dw2[c] = p;
      if (f.db2) f.db2[c] = q;
    } else {
      const float a = f.a ? f.a[c] : 1.f, w = f.w1 ? f.w1[c] : 1.f, b = f.b1 ? f.b1[c] : 0.f;
      if (f.dw1) f.dw1[c] = a * p;
      if (f.db1) f.db1[c] = a * q;
      if (f.da) f.da[c] = f.b1 ? w * p + b * q : w * p;
    }
    return;
  }
  const int k = blockIdx.x - f.n_first, width = f.spc < GATE_MANY ? 1024 : 64, per = (f.cols + width - 1) / width, clip = k / per;
  const int c = (k - clip * per) * width + threadIdx.x % width, step = 1024 / width;
  float s = 0.f;
  if (c < f.cols)
#pragma unroll 8
    for (int w = threadIdx.x / width; w < f.spc; w += step) s += f.gpart[((size_t)clip * f.spc + w) * f.cols + c];
  if (step > 1) {
    __shared__ float share[1024];
    share[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += share[w * 64 + threadIdx.x];
  }
  if (c >= f.cols) return;
  if constexpr (sizeof(T) == 4) ((float*)f.dgate)[(size_t)clip * f.cols + c] = s;
  else ((unsigned short*)f.dgate)[(size_t)clip * f.cols + c] = to_bf16(s);
}

// ---------------------------------------------------------------------------
struct GatedPlan { int lanes, per, rpb, run, spc, workers, blocks, joined; };
// As many waves as a CU holds (backward: half of that, for the registers), each with rows of its own to walk: enough loads in flight (a
// wave holds two rows' worth), and few partial sums.  Above 4096 columns 16 values a lane: with 16 waves of 8 values the backward kernel has half
// the registers and reads the column vectors for every row (8192 x 8192 bf16, both passes 1025 us against 316).
constexpr int FWD_WAVES = 16, BWD_WAVES = 8;
static GatedPlan gated_plan(int rows, int cols, int clip, bool gate, int waves) {
  GatedPlan p;
  p.per = cols <= 4096 ? 8 : 16;
  p.lanes = 8;
  while (p.lanes * p.per < cols) p.lanes *= 2;
  p.rpb = p.lanes >= 256 ? 1 : 256 / p.lanes;
  const int64_t want = (int64_t)device_cus() * waves * 64 / p.lanes;
  const int64_t run = std::max<int64_t>(1, (rows + want - 1) / want), clips = ((int64_t)rows + clip - 1) / clip;
  p.spc = p.joined = 0;
  if (!gate) {
    p.run = (int)run;
    p.workers = (int)((rows + run - 1) / run);
  } else if (clip <= run) {
    p.run = (int)(run / clip * clip);
    p.workers = (int)(((int64_t)rows + p.run - 1) / p.run);
  } else {
    p.spc = (int)((clip + run - 1) / run);
    p.joined = p.spc >= p.rpb;
    if (p.joined) p.spc = (p.spc + p.rpb - 1) / p.rpb * p.rpb;
    p.run = (int)(((int64_t)clip + p.spc - 1) / p.spc);    // at most `run`
    p.workers = (int)(clips * p.spc);                      // at most four times `want`: a clip has more than `run` rows
  }
  p.blocks = (p.workers + p.rpb - 1) / p.rpb;
  return p;
}

size_t gated_norm_workspace(int rows, int cols, int clip) {
  if (rows < 1 || cols < 1 || cols > 8192 || clip < 0) return 0;
  const GatedPlan p = gated_plan(rows, cols, clip ? clip : rows, clip > 0, BWD_WAVES);
  return ((size_t)p.blocks * 4 + (p.joined ? p.blocks : p.spc ? p.workers : 0)) * cols * sizeof(float);
}

template <typename T, int L, int PER, int ACC>
static int run_gated(const GatedArgs& g, const GatedPlan& p, int back, hipStream_t s) {
  constexpr int threads = L > 256 ? L : 256;
  constexpr int lds = PER > 8 ? L * PER * (int)sizeof(float) : 0;         // a column vector
  if (back == 2) {
    if (lds) PT_ENSURE_LDS((gated_norm_bwd_kernel<T, L, PER, ACC, true>), 4 * lds);
    PT_LAUNCH((gated_norm_bwd_kernel<T, L, PER, ACC, true>), dim3(p.blocks), dim3(threads), 4 * lds, s, g);
  } else if (back) {
    if (lds) PT_ENSURE_LDS((gated_norm_bwd_kernel<T, L, PER, ACC, false>), 3 * lds);
    PT_LAUNCH((gated_norm_bwd_kernel<T, L, PER, ACC, false>), dim3(p.blocks), dim3(threads), 3 * lds, s, g);
  } else if (g.layer) PT_LAUNCH((gated_norm_fwd_kernel<T, L, PER, true, ACC>), dim3(p.blocks), dim3(threads), 0, s, g);
  else PT_LAUNCH((gated_norm_fwd_kernel<T, L, PER, false, ACC>), dim3(p.blocks), dim3(threads), 0, s, g);
  return 0;
}
template <typename T, int L, int PER>
static int run_gated(const GatedArgs& g, const GatedPlan& p, Access acc, int back, hipStream_t s) {
  if (acc == ALIGNED) return run_gated<T, L, PER, ALIGNED>(g, p, back, s);
  if constexpr (L == 8)
    if (acc == SCALAR) return run_gated<T, L, PER, SCALAR>(g, p, back, s);
  return run_gated<T, L, PER, ANY>(g, p, back, s);
}
template <typename T>
static int run_gated(const GatedArgs& g, const GatedPlan& p, Access acc, int back, hipStream_t s) {
  switch (p.lanes) {
    case 8: return run_gated<T, 8, 8>(g, p, acc, back, s);
    case 16: return run_gated<T, 16, 8>(g, p, acc, back, s);
    case 32: return run_gated<T, 32, 8>(g, p, acc, back, s);
    case 64: return run_gated<T, 64, 8>(g, p, acc, back, s);
    case 128: return run_gated<T, 128, 8>(g, p, acc, back, s);
    case 256: return run_gated<T, 256, 8>(g, p, acc, back, s);
    default: return p.per == 8 ? run_gated<T, 512, 8>(g, p, acc, back, s) : run_gated<T, 512, 16>(g, p, acc, back, s);
  }
}

static int check_gated(const char* who, const void* x, int64_t ldx, const void* t, int64_t ldt, const void* gate, const float* w1, const float* b1,
                       const float* w2, const float* b2, int64_t rows, int cols, int clip, int kind, int dtype) {
  PT_CHECK(x && rows >= 1 && rows <= 0x7FFFFFFF && cols >= 1 && cols <= 8192, "%s: %lld rows of %d columns (1 to 8192)", who, (long long)rows, cols);
  PT_CHECK(ldx >= cols && (!t || ldt >= cols), "%s: row strides %lld and %lld for %d columns", who, (long long)ldx, (long long)ldt, cols);
  PT_CHECK(!gate || (t && clip >= 1 && rows % clip == 0), "%s: %lld rows in clips of %d", who, (long long)rows, clip);
  PT_CHECK((w1 || !b1) && (w2 || !b2), "%s: a bias comes with its weight", who);
  PT_CHECK((kind == 0 || kind == 1) && (dtype == 0 || dtype == 1), "%s: kind %d, dtype %d", who, kind, dtype);
  return 0;
}
// Two outputs of 64 MB or more together leave the 256 MB of Infinity Cache to x and t, which the backward pass reads again (512 x 88 rows of
// 512 fp32, both passes: 208 -> 192 us; 16,384 x 4096 bf16: 297 -> 287); smaller ones stay in the caches for the next operator
static int gated_stream(const GatedArgs& g, int dtype) { return (int64_t)g.rows * g.cols * (dtype ? 2 : 4) * 2 >= ((int64_t)64 << 20); }
static Access gated_access(const GatedArgs& g, int dtype) {
  const size_t v = dtype ? 8 : 4;
  const uintptr_t p = (uintptr_t)g.x | (uintptr_t)g.t | (uintptr_t)g.gate | (uintptr_t)g.dy | (uintptr_t)g.dh | (uintptr_t)g.y | (uintptr_t)g.h |
                      (uintptr_t)g.dx | (uintptr_t)g.dt | (uintptr_t)g.dgate;
  if ((size_t)g.cols < v) return SCALAR;
  return !(p & 15) && g.cols % v == 0 && g.ldx % v == 0 && (!g.t || g.ldt % v == 0) ? ALIGNED : ANY;
}

int launch_gated_norm_fwd(const void* x, int64_t ldx, const void* t, int64_t ldt, const void* gate, const float* a, const float* w1,
                          const float* b1, const float* w2, const float* b2, void* y, void* h, float* stats, int64_t rows, int cols, int clip,
                          int kind, float eps, int dtype, hipStream_t s) {
  if (check_gated("gated_norm_fwd", x, ldx, t, ldt, gate, w1, b1, w2, b2, rows, cols, clip, kind, dtype)) return 1;
  PT_CHECK((t || w2) && (!t || y) && (!w2 || h) && ((uintptr_t)stats & 15) == 0, "gated_norm_fwd: null or misaligned argument");
  GatedArgs g = {};
  g.x = x; g.t = t; g.gate = gate; g.a = a; g.w1 = w1; g.b1 = b1; g.w2 = w2; g.b2 = b2; g.y = y; g.h = h; g.stats = stats;
  g.ldx = (size_t)ldx; g.ldt = (size_t)ldt; g.rows = (int)rows; g.cols = cols; g.clip = gate ? clip : (int)rows; g.eps = eps;
  const GatedPlan p = gated_plan(g.rows, cols, g.clip, gate != nullptr, FWD_WAVES);
  g.run = p.run; g.spc = p.spc;
  g.layer = kind == 0;
  g.stream = gated_stream(g, dtype);
  const Access acc = gated_access(g, dtype);
  return dtype ? run_gated<unsigned short>(g, p, acc, 0, s) : run_gated<float>(g, p, acc, 0, s);
}

int launch_gated_norm_bwd(const void* x, int64_t ldx, const void* t, int64_t ldt, const void* gate, const float* a, const float* w1,
                          const float* b1, const float* w2, const float* stats, const void* dy, const void* dh, void* dx, void* dt,
                          void* dgate, float* da, float* dw1, float* db1, float* dw2, float* db2, void* ws, size_t ws_bytes, int64_t rows,
                          int cols, int clip, int kind, int dtype, hipStream_t s) {
  if (check_gated("gated_norm_bwd", x, ldx, t, ldt, gate, w1, b1, w2, nullptr, rows, cols, clip, kind, dtype)) return 1;
  PT_CHECK(stats && dx && (dy || dh) && (!dh || w2) && (!dgate || gate) && (!dt || t), "gated_norm_bwd: null argument");
  PT_CHECK(ws && ws_bytes >= gated_norm_workspace((int)rows, cols, gate ? clip : 0) && (((uintptr_t)ws | (uintptr_t)stats) & 15) == 0,
           "gated_norm_bwd: workspace of %zu bytes, %zu needed, 16-byte aligned", ws_bytes, gated_norm_workspace((int)rows, cols, gate ? clip : 0));
  if (!t) a = w1 = b1 = nullptr;                           // y is x, whatever else is given
  GatedArgs g = {};
  g.x = x; g.t = t; g.gate = gate; g.a = a; g.w1 = w1; g.b1 = b1; g.w2 = w2; g.dy = dy; g.dh = dh; g.stats = const_cast<float*>(stats);
  g.dx = dx; g.dt = dt; g.dgate = dgate;
  g.ldx = (size_t)ldx; g.ldt = (size_t)ldt; g.rows = (int)rows; g.cols = cols; g.clip = gate ? clip : (int)rows;
  const GatedPlan p = gated_plan(g.rows, cols, g.clip, gate != nullptr, BWD_WAVES);
  g.run = p.run; g.spc = p.spc;
  g.part = (float*)ws;
  g.gpart = p.spc && dgate ? g.part + (size_t)p.blocks * 4 * cols : nullptr;
  g.joined = p.joined && dgate;
  g.layer = kind == 0;
  g.stream = gated_stream(g, dtype);
  const Access acc = gated_access(g, dtype);
  const int bias = b1 || db1 || db2 ? 1 : 0;
  if (dtype ? run_gated<unsigned short>(g, p, acc, 1 + bias, s) : run_gated<float>(g, p, acc, 1 + bias, s)) return 1;
  GatedFinish f = {};
  f.part = g.part; f.gpart = g.gpart; f.a = a; f.w1 = w1; f.b1 = b1;
  f.da = t ? da : nullptr; f.dw1 = t ? dw1 : nullptr; f.db1 = t ? db1 : nullptr; f.dw2 = dw2; f.db2 = db2;
  f.dgate = dgate; f.blocks = p.blocks; f.cols = cols; f.spc = p.joined ? p.spc / p.rpb : p.spc;
  f.col_blocks = (cols + 63) / 64;
  f.n_first = 2 * f.col_blocks;
  const int width = f.spc < GATE_MANY ? 1024 : 64;
  const int64_t gate_blocks = g.gpart ? (int64_t)(rows / clip) * ((cols + width - 1) / width) : 0;
  PT_CHECK(f.n_first + gate_blocks < 0x7FFFFFFF, "gated_norm_bwd: too many clips");
  if (dtype) PT_LAUNCH(gated_norm_finish_kernel<unsigned short>, dim3((unsigned)(f.n_first + gate_blocks)), dim3(1024), 0, s, f);
  else PT_LAUNCH(gated_norm_finish_kernel<float>, dim3((unsigned)(f.n_first + gate_blocks)), dim3(1024), 0, s, f);
  return 0;
}

}  // namespace pt
