// Attention over a window of keys and a few first ones (sinks), forward, backward and for single tokens over a cache.
//
//   row i of a sequence stands at position t = i + (Nk - Nq); key j is visible to it where
//     j <= t + right  and  (j >= t - left  or  j < sinks)  and  j < length
//   o_i = sum_j p_ij v_j,  p_i = softmax over the visible j of scale q_i.k_j;  a row that sees nothing gives 0
//   backward, with P from the kept log-sum-exp and delta_i = do_i.o_i:
//     dV = P^T dO,  dS = P (dO V^T - delta) scale,  dQ = dS K,  dK = dS^T Q      (dK, dV summed over the query heads of a group)
//
// Bound by the matrix cores (4 D flops a visible pair forward, 14 D backward: S and dP are computed in both of its kernels, which
// costs 4 D and saves the atomics or the round trip of dQ) and, next to them, by the exponentials on the vector unit.
//
// Layout.  All products are 32 x 32 tiles with 16 contraction steps: bf16 one v_mfma_f32_32x32x16_bf16, fp32 eight
// v_mfma_f32_32x32x2_f32 on the same lanes (element e of a lane's eight is contraction step 8 (lane / 32) + e in both, so one code
// serves both types).  A result tile has its column in the lane and its rows in registers: element r is row
// (r & 3) + 8 (r >> 2) + 4 (lane / 32).  Scores are always taken so that what follows is the SECOND operand of the next product with
// exactly these registers (its contraction order being 4 + 4 rows per lane half): S^T = K Q^T then O^T += V^T P^T, and in the dK / dV
// kernel S = Q K^T then dV^T += dO^T P: probabilities never leave the registers, softmax statistics are one value per lane.
// The first operand of those second products is the transpose of a tile that lies row by row in LDS: bf16 reads it with the
// transposing ds_read_b64_tr_b16, fp32 with single words.  LDS rows hold 16-byte chunks in an order that is free of bank conflicts
// for both kinds of reads: chunk ^= bit-reversed low bits of the row.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "pt_common.h"

namespace pt {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_t;

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct Types;
template <> struct Types<__bf16> { typedef bf16x8 frag; typedef bf16x4 quad; };
template <> struct Types<float> { typedef f32x8 frag; typedef f32x4 quad; };

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}
// the sum / maximum over the two lanes that share a column
__device__ __forceinline__ float half_other(float v) {
  const unsigned w = __builtin_bit_cast(unsigned, v);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  const unsigned b0 = b[0], b1 = b[1];
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? b0 : b1);
}

struct WinArgs {
  const void* q; const void* k; const void* v;
  void* o; float* lse;                                   // lse [B][H][Nq], in powers of two; +inf for a row that sees nothing
  const void* od; const void* dod;                       // backward: o and its gradient, (B, Nq, H, D)
  void* dq; void* dk; void* dv; float* delta;            // delta [B][H][Nq]
  float* part;                                           // shares of the first keys' gradients (see win_bwd_sink_kernel)
  int64_t sq[3], sk[3], sv[3];                           // strides of batch, row, head in values
  const int* lengths;
  int B, Nq, Nk, H, Hk, D, left, right, sinks;
  float sc, scale;                                       // scale * log2(e), scale
  int far, far_chunks, far_rows;                         // first row index that sees the first keys only as sinks, its chunks, rows of one
};

__device__ __forceinline__ int length_of(const WinArgs& a, int b) { return a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk; }
__device__ __forceinline__ bool visible(const WinArgs& a, int len, int t, int j) {
  return j <= t + a.right && (j >= t - a.left || j < a.sinks) && j < len;
}

// LDS image of a tile: rows of DP values, 16-byte chunks permuted within the row
template <typename T, int DP>
struct Tile {
  static constexpr int RB = DP * (int)sizeof(T), CPR = RB / 16, EPC = 16 / (int)sizeof(T);
  typedef typename Types<T>::frag frag;
  // 128-byte rows: two rows per turn of the banks, so the row's lowest bit is a half already
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (RB == 128) return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
    else return (row & 1) << 3 | (row & 2) << 1 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swz(row)) << 4); }
  // 8 values along the row: columns 16 s + 8 h .. + 7 of row
  static __device__ __forceinline__ frag row_frag(const unsigned char* m, int row, int s, int h) {
    if constexpr (sizeof(T) == 2) return *reinterpret_cast<const bf16x8*>(m + at(row, 2 * s + h));
    else {
      const f32x4 x = *reinterpret_cast<const f32x4*>(m + at(row, 4 * s + 2 * h)), y = *reinterpret_cast<const f32x4*>(m + at(row, 4 * s + 2 * h + 1));
      const frag f = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      return f;
    }
  }
  // 8 values down a column: rows row0 + 8 (e >> 2) + 4 h + (e & 3) of column 32 db + lane % 32
  static __device__ __forceinline__ frag col_frag(const unsigned char* m, int row0, int db, int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int tq = (lane >> 2) & 3, tp = lane & 3, tg = (lane >> 4) & 1, c = db * 4 + tg * 2 + (tp >> 1);
      const int r0 = row0 + 4 * h + tq, r1 = r0 + 8;
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(m + at(r0, c) + (tp & 1) * 8));
      const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(m + at(r1, c) + (tp & 1) * 8));
      const s16x8 f = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      return __builtin_bit_cast(bf16x8, f);
    } else {
      const int d = db * 32 + (lane & 31);
      frag f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = row0 + 8 * (e >> 2) + 4 * h + (e & 3);
        f[e] = *reinterpret_cast<const float*>(m + at(r, d / 4) + (d & 3) * 4);
      }
      return f;
    }
  }
};

// R rows of a tile on their way from memory to LDS; rows from `limit` on and columns from D on are zeros
template <typename T, int DP, int R>
struct Stage {
  typedef Tile<T, DP> tile;
  static constexpr int N = R * tile::CPR / 256;
  static_assert(N >= 1, "tile too small for the workgroup");
  u32x4 x[N];
  __device__ __forceinline__ void load(const T* __restrict__ base, int64_t stride, int row0, int limit, int D) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = threadIdx.x + 256 * i, row = row0 + e / tile::CPR, c = (e % tile::CPR) * tile::EPC;
      x[i] = u32x4{0u, 0u, 0u, 0u};
      if (row >= 0 && row < limit && c < D) x[i] = *reinterpret_cast<const u32x4*>(base + row * stride + c);
    }
  }
  __device__ __forceinline__ void store(unsigned char* m) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = threadIdx.x + 256 * i;
      *reinterpret_cast<u32x4*>(m + tile::at(e / tile::CPR, e % tile::CPR)) = x[i];
    }
  }
};

// 8 values of row `row` from memory, as an operand
template <typename T>
__device__ __forceinline__ typename Types<T>::frag global_frag(const T* __restrict__ base, int64_t stride, int row, int limit, int c, int D) {
  typename Types<T>::frag f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (T)0.f;
  if (row < limit && c < D) f = *reinterpret_cast<const typename Types<T>::frag*>(base + row * stride + c);
  return f;
}
template <typename T>
__device__ __forceinline__ typename Types<T>::frag pack(const f32x16& p, int s2) {
  typename Types<T>::frag f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (T)p[8 * s2 + e];
  return f;
}
// a transposed result (lane: row `row` of the output, registers: columns) times x
template <typename T, int DP>
__device__ __forceinline__ void store_transposed(T* __restrict__ base, const f32x16 (&acc)[DP / 32], int h, int D, float x) {
  typedef typename Types<T>::quad quad;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = db * 32 + 8 * g + 4 * h;
      if (c < D) {
        const quad o = {(T)(acc[db][4 * g] * x), (T)(acc[db][4 * g + 1] * x), (T)(acc[db][4 * g + 2] * x), (T)(acc[db][4 * g + 3] * x)};
        *reinterpret_cast<quad*>(base + c) = o;
      }
    }
}

// Key tiles of KT that rows at positions [t0, t1] may see: [0, first) for the sinks, then [from, to)
template <int KT>
__device__ __forceinline__ void key_tiles(const WinArgs& a, int len, int t0, int t1, int& first, int& from, int& to) {
  const int hi = min(t1 + a.right, len - 1), lo = max(t0 - a.left, 0);
  first = (min(a.sinks, hi + 1) + KT - 1) / KT;
  if (hi < 0) first = 0;
  from = max(lo / KT, first);
  to = hi < lo ? from : max(hi / KT + 1, from);
}

// ---------------------------------------------------------------------------
// Forward: 4 waves of 32 rows each over common key tiles
// ---------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void win_fwd_kernel(const WinArgs a) {
  constexpr int KT = sizeof(T) == 2 ? 64 : 32, NB = KT / 32;
  typedef Tile<T, DP> tile;
  __shared__ __attribute__((aligned(1024))) unsigned char Ks[KT * tile::RB], Vs[KT * tile::RB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
  const int head = blockIdx.y, b = blockIdx.z, kvh = head / (a.H / a.Hk);
  const int len = length_of(a, b), shift = a.Nk - a.Nq;
  const int i0 = blockIdx.x * 128 + wave * 32, row = i0 + col, t = row + shift;
  const T* __restrict__ K = (const T*)a.k + b * a.sk[0] + kvh * a.sk[2];
  const T* __restrict__ V = (const T*)a.v + b * a.sv[0] + kvh * a.sv[2];
  const T* __restrict__ Q = (const T*)a.q + b * a.sq[0] + head * a.sq[2];
  typename Types<T>::frag qf[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) qf[s] = global_frag(Q, a.sq[1], row, a.Nq, 16 * s + 8 * h, a.D);
  f32x16 o[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) o[db] = zero16();
  float m = -INFINITY, l = 0.f;
  int first, from, to;
  const int T0 = blockIdx.x * 128 + shift, T1 = min(blockIdx.x * 128 + 127, a.Nq - 1) + shift;
  key_tiles<KT>(a, len, T0, T1, first, from, to);
  const int tiles = first + (to - from);
  const int w0 = i0 + shift, w1 = min(i0 + 31, a.Nq - 1) + shift;        // positions of this wave
  Stage<T, DP, KT> sk, sv;
  if (tiles > 0) {
    const int k0 = (first ? 0 : from) * KT;
    sk.load(K, a.sk[1], k0, len, a.D);
    sv.load(V, a.sv[1], k0, len, a.D);
  }
  for (int n = 0; n < tiles; ++n) {
    const int k0 = (n < first ? n : from + n - first) * KT, k1 = k0 + KT - 1;
    __syncthreads();
    sk.store(Ks);
    sv.store(Vs);
    __syncthreads();
    if (n + 1 < tiles) {
      const int kn = (n + 1 < first ? n + 1 : from + n + 1 - first) * KT;
      sk.load(K, a.sk[1], kn, len, a.D);
      sv.load(V, a.sv[1], kn, len, a.D);
    }
    if (i0 >= a.Nq || k0 > w1 + a.right || (k1 < w0 - a.left && k0 >= a.sinks)) continue;
    f32x16 st[NB];
#pragma unroll
    for (int x = 0; x < NB; ++x) {
      st[x] = zero16();
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) st[x] = mma(tile::row_frag(Ks, 32 * x + col, s, h), qf[s], st[x]);
    }
    if (!(k1 <= w0 + a.right && k1 < len && (k0 >= w1 - a.left || k1 < a.sinks))) {
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          st[x][r] = visible(a, len, t, k0 + 32 * x + (r & 3) + 8 * (r >> 2) + 4 * h) ? st[x][r] : -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < NB; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[x][r]);
    mx = fmaxf(mx, half_other(mx)) * a.sc;
    const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn;    // nothing visible so far: every exponential is 0
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < NB; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        st[x][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[x][r], a.sc, -base));
        sum += st[x][r];
      }
    l = l * alpha + sum;                                                 // this lane's half of the column; joined at the end
    m = mn;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
#pragma unroll
    for (int x = 0; x < NB; ++x)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const auto pf = pack<T>(st[x], s2);                              // probabilities in [0, 1] to bf16: 2^-9 of each
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) o[db] = mma(tile::col_frag(Vs, 32 * x + 16 * s2, db, lane), pf, o[db]);
      }
  }
  if (row >= a.Nq) return;
  l += half_other(l);
  store_transposed<T, DP>((T*)a.o + (((int64_t)b * a.Nq + row) * a.H + head) * a.D, o, h, a.D, l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l));
  if (a.lse && h == 0) a.lse[((int64_t)b * a.H + head) * a.Nq + row] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// ---------------------------------------------------------------------------
// Backward, dQ (and delta): rows and key tiles as forward
// ---------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void win_bwd_q_kernel(const WinArgs a) {
  constexpr int KT = sizeof(T) == 2 ? 64 : 32, NB = KT / 32;
  typedef Tile<T, DP> tile;
  __shared__ __attribute__((aligned(1024))) unsigned char Ks[KT * tile::RB], Vs[KT * tile::RB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
  const int head = blockIdx.y, b = blockIdx.z, kvh = head / (a.H / a.Hk);
  const int len = length_of(a, b), shift = a.Nk - a.Nq;
  const int i0 = blockIdx.x * 128 + wave * 32, row = i0 + col, t = row + shift;
  const T* __restrict__ K = (const T*)a.k + b * a.sk[0] + kvh * a.sk[2];
  const T* __restrict__ V = (const T*)a.v + b * a.sv[0] + kvh * a.sv[2];
  const T* __restrict__ Q = (const T*)a.q + b * a.sq[0] + head * a.sq[2];
  const int64_t so = (int64_t)a.H * a.D, ob = ((int64_t)b * a.Nq * a.H + head) * a.D;
  typename Types<T>::frag qf[DP / 16], gf[DP / 16];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    qf[s] = global_frag(Q, a.sq[1], row, a.Nq, 16 * s + 8 * h, a.D);
    gf[s] = global_frag((const T*)a.dod + ob, so, row, a.Nq, 16 * s + 8 * h, a.D);
    const auto of = global_frag((const T*)a.od + ob, so, row, a.Nq, 16 * s + 8 * h, a.D);
#pragma unroll
    for (int e = 0; e < 8; ++e) delta += (float)gf[s][e] * (float)of[e];
  }
  delta += half_other(delta);
  const int64_t li = ((int64_t)b * a.H + head) * a.Nq + row;
  const float lse = row < a.Nq ? a.lse[li] : INFINITY;
  if (row < a.Nq && h == 0) a.delta[li] = delta;
  f32x16 dq[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) dq[db] = zero16();
  int first, from, to;
  const int T0 = blockIdx.x * 128 + shift, T1 = min(blockIdx.x * 128 + 127, a.Nq - 1) + shift;
  key_tiles<KT>(a, len, T0, T1, first, from, to);
  const int tiles = first + (to - from);
  const int w0 = i0 + shift, w1 = min(i0 + 31, a.Nq - 1) + shift;
  Stage<T, DP, KT> sk, sv;
  if (tiles > 0) {
    const int k0 = (first ? 0 : from) * KT;
    sk.load(K, a.sk[1], k0, len, a.D);
    sv.load(V, a.sv[1], k0, len, a.D);
  }
  for (int n = 0; n < tiles; ++n) {
    const int k0 = (n < first ? n : from + n - first) * KT, k1 = k0 + KT - 1;
    __syncthreads();
    sk.store(Ks);
    sv.store(Vs);
    __syncthreads();
    if (n + 1 < tiles) {
      const int kn = (n + 1 < first ? n + 1 : from + n + 1 - first) * KT;
      sk.load(K, a.sk[1], kn, len, a.D);
      sv.load(V, a.sv[1], kn, len, a.D);
    }
    if (i0 >= a.Nq || k0 > w1 + a.right || (k1 < w0 - a.left && k0 >= a.sinks)) continue;
    const bool all = k1 <= w0 + a.right && k1 < len && (k0 >= w1 - a.left || k1 < a.sinks);
#pragma unroll
    for (int x = 0; x < NB; ++x) {
      f32x16 st = zero16(), dp = zero16();
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        st = mma(tile::row_frag(Ks, 32 * x + col, s, h), qf[s], st);
        dp = mma(tile::row_frag(Vs, 32 * x + col, s, h), gf[s], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], a.sc, -lse)), ds = p * (dp[r] - delta);
        st[r] = all || visible(a, len, t, k0 + 32 * x + (r & 3) + 8 * (r >> 2) + 4 * h) ? ds : 0.f;
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const auto df = pack<T>(st, s2);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) dq[db] = mma(tile::col_frag(Ks, 32 * x + 16 * s2, db, lane), df, dq[db]);
      }
    }
  }
  if (row < a.Nq) store_transposed<T, DP>((T*)a.dq + (((int64_t)b * a.Nq + row) * a.H + head) * a.D, dq, h, a.D, a.scale);
}

// ---------------------------------------------------------------------------
// Backward, dK and dV: 4 waves of 32 keys each over common tiles of 32 rows, all query heads of the group in turn.
// SINK: the rows far behind the window, which see the first 32-key blocks as sinks only.  There are as many of these rows as the
// sequence is long and only a few keys, so the four waves take the SAME keys and a quarter of the rows each, the rows are cut
// into chunks, and every wave leaves its share in fp32; win_bwd_join_kernel adds the shares in order.
// ---------------------------------------------------------------------------
template <typename T, int DP, bool SINK>
__global__ __launch_bounds__(256, DP * (int)sizeof(T) <= 128 ? 2 : 1) void win_bwd_kv_kernel(const WinArgs a) {
  constexpr int QT = SINK ? 128 : 32;
  typedef Tile<T, DP> tile;
  extern __shared__ __attribute__((aligned(1024))) unsigned char win_smem[];
  unsigned char* Qs = win_smem;
  unsigned char* Gs = Qs + QT * tile::RB;
  float* ls = reinterpret_cast<float*>(Gs + QT * tile::RB);
  float* ds_ = ls + QT;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
  const int group = a.H / a.Hk, shift = a.Nk - a.Nq, b = blockIdx.z;
  const int blocks = (a.sinks + 31) / 32;                                // of 32 first keys
  const int kvh = SINK ? blockIdx.y / group : blockIdx.y;
  const int len = length_of(a, b);
  const int k0 = SINK ? (blockIdx.x % blocks) * 32 : blockIdx.x * 128 + wave * 32, key = k0 + col;
  const T* __restrict__ K = (const T*)a.k + b * a.sk[0] + kvh * a.sk[2];
  const T* __restrict__ V = (const T*)a.v + b * a.sv[0] + kvh * a.sv[2];
  typename Types<T>::frag kf[DP / 16], vf[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    kf[s] = global_frag(K, a.sk[1], key, len, 16 * s + 8 * h, a.D);
    vf[s] = global_frag(V, a.sv[1], key, len, 16 * s + 8 * h, a.D);
  }
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) { dk[db] = zero16(); dv[db] = zero16(); }
  // rows that this workgroup looks at
  int r0, r1;
  if constexpr (SINK) {
    r0 = a.far + (blockIdx.x / blocks) * a.far_rows;
    r1 = min(r0 + a.far_rows, a.Nq);
  } else {
    const int kb = blockIdx.x * 128;
    r0 = max(kb - a.right - shift, 0) / QT * QT;
    r1 = kb >= len ? 0 : (int)min((int64_t)kb + 127 + a.left - shift + 1, (int64_t)a.Nq);
  }
  const int per = r1 > r0 ? (r1 - r0 + QT - 1) / QT : 0, total = SINK ? per : per * group;
  const int64_t so = (int64_t)a.H * a.D;
  Stage<T, DP, QT> sq, sg;
  float nl = INFINITY, nd = 0.f;
  auto fetch = [&](int n) {
    const int head = SINK ? (int)blockIdx.y : kvh * group + n / per, rr = r0 + (n % per) * QT;
    sq.load((const T*)a.q + b * a.sq[0] + head * a.sq[2], a.sq[1], rr, a.Nq, a.D);
    sg.load((const T*)a.dod + ((int64_t)b * a.Nq * a.H + head) * a.D, so, rr, a.Nq, a.D);
    if (threadIdx.x < QT) {
      const int i = rr + threadIdx.x;
      const int64_t li = ((int64_t)b * a.H + head) * a.Nq + i;
      nl = i < r1 ? a.lse[li] : INFINITY;                                // a row of no weight
      nd = i < r1 ? a.delta[li] : 0.f;
    }
  };
  if (total > 0) fetch(0);
  for (int n = 0; n < total; ++n) {
    __syncthreads();
    sq.store(Qs);
    sg.store(Gs);
    if (threadIdx.x < QT) { ls[threadIdx.x] = nl; ds_[threadIdx.x] = nd; }
    __syncthreads();
    if (n + 1 < total) fetch(n + 1);
    const int sub = SINK ? wave * 32 : 0, t0 = r0 + (n % per) * QT + sub + shift, t1 = t0 + 31;
    if (k0 > t1 + a.right || (k0 + 31 < t0 - a.left && k0 >= a.sinks) || k0 >= len) continue;
    const bool all = k0 + 31 <= t0 + a.right && k0 + 31 < len && (k0 >= t1 - a.left || k0 + 31 < a.sinks);
    f32x16 st = zero16(), dp = zero16();
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      st = mma(tile::row_frag(Qs, sub + col, s, h), kf[s], st);
      dp = mma(tile::row_frag(Gs, sub + col, s, h), vf[s], dp);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 L4 = *reinterpret_cast<const f32x4*>(ls + sub + 8 * g + 4 * h), D4 = *reinterpret_cast<const f32x4*>(ds_ + sub + 8 * g + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * g + e;
        const bool on = all || visible(a, len, t0 + 8 * g + 4 * h + e, key);
        const float p = on ? __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], a.sc, -L4[e])) : 0.f;
        dp[r] = on ? p * (dp[r] - D4[e]) : 0.f;
        st[r] = p;
      }
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      const auto pf = pack<T>(st, s2);
      const auto df = pack<T>(dp, s2);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) {
        dv[db] = mma(tile::col_frag(Gs, sub + 16 * s2, db, lane), pf, dv[db]);
        dk[db] = mma(tile::col_frag(Qs, sub + 16 * s2, db, lane), df, dk[db]);
      }
    }
  }
  if constexpr (SINK) {
    if (key >= a.sinks) return;
    // share [slot][b][kvh][2][sinks][D]; slot 0 is the window's part
    const int slot = 1 + ((blockIdx.x / blocks) * group + blockIdx.y % group) * 4 + wave;
    float* out = a.part + ((((int64_t)slot * a.B + b) * a.Hk + kvh) * 2 * a.sinks + key) * a.D;
    store_transposed<float, DP>(out, dk, h, a.D, a.scale);
    store_transposed<float, DP>(out + (int64_t)a.sinks * a.D, dv, h, a.D, 1.f);
  } else {
    if (key >= a.Nk) return;
    if (a.part && key < a.sinks) {
      float* out = a.part + (((int64_t)b * a.Hk + kvh) * 2 * a.sinks + key) * a.D;
      store_transposed<float, DP>(out, dk, h, a.D, a.scale);
      store_transposed<float, DP>(out + (int64_t)a.sinks * a.D, dv, h, a.D, 1.f);
    } else {
      const int64_t at = (((int64_t)b * a.Nk + key) * a.Hk + kvh) * a.D;
      store_transposed<T, DP>((T*)a.dk + at, dk, h, a.D, a.scale);
      store_transposed<T, DP>((T*)a.dv + at, dv, h, a.D, 1.f);
    }
  }
}

// the first keys' gradients: the shares in order
template <typename T>
__global__ __launch_bounds__(256) void win_bwd_join_kernel(const WinArgs a, int slots) {
  const int64_t n = (int64_t)a.B * a.Hk * 2 * a.sinks * a.D, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < slots; ++k) s += a.part[k * n + i];
  int64_t r = i;
  const int d = (int)(r % a.D); r /= a.D;
  const int key = (int)(r % a.sinks); r /= a.sinks;
  const int which = (int)(r & 1); r >>= 1;
  const int kvh = (int)(r % a.Hk), b = (int)(r / a.Hk);
  ((T*)(which ? a.dv : a.dk))[(((int64_t)b * a.Nk + key) * a.Hk + kvh) * a.D + d] = (T)s;
}

// ---------------------------------------------------------------------------
// One token: scores of G query heads of a group against the visible keys of a slice of the cache.  Bound by HBM (every visible key
// and value is read once for all heads of the group), so it runs on the vector unit straight from memory: L lanes hold a key's
// row (8 values each), the wave's 64 / L lane groups walk keys side by side, each with its own running maximum and sum, joined at
// the end.  Few sequences: the visible keys are cut into slices, joined by a second kernel.
// ---------------------------------------------------------------------------
struct StepArgs {
  const void* q; const void* k; const void* v; void* o; const int* lengths;
  int64_t sq[2], sk[3], sv[3];                           // q: batch, head; caches: batch, row, head
  int B, N, H, Hk, D, left, sinks, splits;
  float sc;
  float* part;                                           // [B][H][splits][D + 2]: unnormalised output, maximum, sum
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool on, float (&x)[8]) {
  typename Types<T>::frag f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (T)0.f;
  if (on) f = *reinterpret_cast<const typename Types<T>::frag*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)f[e];
}

template <typename T, int L, int G>
__global__ __launch_bounds__(256) void win_step_kernel(const StepArgs a) {
  constexpr int KW = 64 / L, U = 4;                      // keys side by side in a wave, and turns whose loads go out together
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane % L, sub = lane / L;
  const int groups = (a.H / a.Hk + G - 1) / G;
  const int split = blockIdx.x, kvh = blockIdx.y / groups, g0 = (blockIdx.y % groups) * G, b = blockIdx.z;
  const int group = a.H / a.Hk, heads = min(G, group - g0), h0 = kvh * group + g0;
  const int len = min(max(a.lengths[b], 0), a.N), t = len - 1;
  // the visible keys in order: [0, ns) sinks, then [lo, len)
  const int lo = max(t - a.left, 0), ns = min(min(a.sinks, lo), len), seen = len > 0 ? ns + (len - lo) : 0;
  const int per = (seen + a.splits - 1) / a.splits, n0 = min(split * per, seen), n1 = min(n0 + per, seen);
  const T* __restrict__ K = (const T*)a.k + b * a.sk[0] + kvh * a.sk[2] + li * 8;
  const T* __restrict__ V = (const T*)a.v + b * a.sv[0] + kvh * a.sv[2] + li * 8;
  const bool in = li * 8 < a.D;
  float q[G][8], acc[G][8], m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    load8((const T*)a.q + b * a.sq[0] + (h0 + min(g, heads - 1)) * a.sq[1] + li * 8, in, q[g]);
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) { q[g][e] *= a.sc; acc[g][e] = 0.f; }
  }
  for (int n = n0 + wave * KW * U; n < n1; n += 4 * KW * U) {
    float k[U][8], v[U][8];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = n + u * KW + sub;
      on[u] = i < n1;
      const int j = i < ns ? i : lo + i - ns;
      load8(K + (on[u] ? j : 0) * a.sk[1], on[u] && in, k[u]);
      load8(V + (on[u] ? j : 0) * a.sv[1], on[u] && in, v[u]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float s[U], mx = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf(q[g][e], k[u][e], d);
#pragma unroll
        for (int x = 1; x < L; x <<= 1) d += __shfl_xor(d, x);
        s[u] = on[u] ? d : -INFINITY;
        mx = fmaxf(mx, s[u]);
      }
      const float base = mx == -INFINITY ? 0.f : mx, alpha = __builtin_amdgcn_exp2f(m[g] - base);
      m[g] = mx;
      l[g] *= alpha;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[g][e] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = __builtin_amdgcn_exp2f(s[u] - base);
        l[g] += p;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[g][e] = fmaf(p, v[u][e], acc[g][e]);
      }
    }
  }
  // join the lane groups, then the waves
  __shared__ float red[4][G][L * 8 + 2];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float top = m[g];
#pragma unroll
    for (int x = L; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float w = __builtin_amdgcn_exp2f(m[g] - (top == -INFINITY ? 0.f : top));
    l[g] *= w;
#pragma unroll
    for (int x = L; x < 64; x <<= 1) l[g] += __shfl_xor(l[g], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      acc[g][e] *= w;
#pragma unroll
      for (int x = L; x < 64; x <<= 1) acc[g][e] += __shfl_xor(acc[g][e], x);
      if (sub == 0) red[wave][g][li * 8 + e] = acc[g][e];
    }
    if (lane == 0) { red[wave][g][L * 8] = top; red[wave][g][L * 8 + 1] = l[g]; }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < heads * L * 8; x += 256) {
    const int g = x / (L * 8), d = x % (L * 8);
    if (d >= a.D) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, red[w][g][L * 8]);
    const float base = top == -INFINITY ? 0.f : top;
    float s = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(red[w][g][L * 8] - base);
      s += f * red[w][g][L * 8 + 1];
      y += f * red[w][g][d];
    }
    const int64_t oh = (int64_t)b * a.H + h0 + g;
    if (a.splits == 1) {
      ((T*)a.o)[oh * a.D + d] = (T)(s == 0.f ? 0.f : y / s);
    } else {
      float* out = a.part + (oh * a.splits + split) * (a.D + 2);
      out[d] = y;
      if (d == 0) { out[a.D] = top; out[a.D + 1] = s; }
    }
  }
}
template <typename T>
__global__ __launch_bounds__(128) void win_step_join_kernel(const StepArgs a) {
  const int64_t oh = blockIdx.x;
  const int d = threadIdx.x;
  if (d >= a.D) return;
  const float* p = a.part + oh * a.splits * (a.D + 2);
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, p[s * (a.D + 2) + a.D]);
  const float base = top == -INFINITY ? 0.f : top;
  float l = 0.f, y = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float f = __builtin_amdgcn_exp2f(p[s * (a.D + 2) + a.D] - base);
    l += f * p[s * (a.D + 2) + a.D + 1];
    y += f * p[s * (a.D + 2) + d];
  }
  ((T*)a.o)[oh * a.D + d] = (T)(l == 0.f ? 0.f : y / l);
}

// ---------------------------------------------------------------------------
constexpr int WIN_FAR = 1 << 29, WIN_MAX = 1 << 28;

static int check_win(const char* who, int B, int Nq, int Nk, int H, int Hk, int D, int left, int right, int sinks, float scale, int dtype) {
  PT_CHECK(B >= 1 && B <= 65535 && Nq >= 1 && Nk >= Nq && Nk <= WIN_MAX, "%s: %d sequences of %d rows and %d keys", who, B, Nq, Nk);
  PT_CHECK(H >= 1 && H <= 65535 && Hk >= 1 && H % Hk == 0, "%s: %d query heads over %d key heads", who, H, Hk);
  PT_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "%s: head dimension %d (a multiple of 8 up to 128)", who, D);
  PT_CHECK(left >= -1 && right >= -1 && sinks >= 0 && sinks <= 128, "%s: window of %d left, %d right, %d first keys (up to 128)", who, left, right, sinks);
  PT_CHECK(scale > 0.f && scale < INFINITY && (dtype == 0 || dtype == 1), "%s: scale %g, dtype %d", who, scale, dtype);
  return 0;
}
// 16-byte loads: addresses and strides in multiples of 16 bytes
static bool aligned16(const void* p, const int64_t* s, int n, int dtype) {
  const int64_t v = dtype ? 8 : 4;
  bool ok = !((uintptr_t)p & 15);
  for (int i = 0; i < n; ++i) ok = ok && s[i] % v == 0;
  return ok;
}
static WinArgs win_args(const void* q, const void* k, const void* v, const int64_t* st, const int* lengths, int B, int Nq, int Nk, int H, int Hk, int D,
                        int left, int right, int sinks, float scale) {
  WinArgs a = {};
  a.q = q; a.k = k; a.v = v; a.lengths = lengths;
  for (int i = 0; i < 3; ++i) { a.sq[i] = st[i]; a.sk[i] = st[3 + i]; a.sv[i] = st[6 + i]; }
  a.B = B; a.Nq = Nq; a.Nk = Nk; a.H = H; a.Hk = Hk; a.D = D;
  a.left = left < 0 || left > WIN_FAR ? WIN_FAR : left;
  a.right = right < 0 || right > WIN_FAR ? WIN_FAR : right;
  a.sinks = std::min(sinks, Nk);
  a.scale = scale; a.sc = scale * LOG2E;
  // rows behind the window of the first 128 keys, which see the sinks among those as sinks only
  const int64_t far = std::max<int64_t>((int64_t)128 + a.left - (Nk - Nq), 0);
  if (a.sinks > 0 && far < Nq) {
    a.far = (int)far;
    const int rows = Nq - a.far, want = std::max(1, 1024 / (B * H));       // about four workgroups per CU
    a.far_rows = std::max(512, ((rows + want - 1) / want + 127) / 128 * 128);
    a.far_chunks = (rows + a.far_rows - 1) / a.far_rows;
  }
  return a;
}

template <typename T, int DP>
static int run_win_fwd(const WinArgs& a, hipStream_t s) {
  PT_LAUNCH((win_fwd_kernel<T, DP>), dim3((a.Nq + 127) / 128, a.H, a.B), dim3(256), 0, s, a);
  return 0;
}
template <typename T, int DP>
static int run_win_bwd(const WinArgs& a, hipStream_t s) {
  constexpr int lds = 2 * 32 * Tile<T, DP>::RB + 2 * 32 * 4, lds_sink = 2 * 128 * Tile<T, DP>::RB + 2 * 128 * 4;
  PT_LAUNCH((win_bwd_q_kernel<T, DP>), dim3((a.Nq + 127) / 128, a.H, a.B), dim3(256), 0, s, a);
  PT_LAUNCH((win_bwd_kv_kernel<T, DP, false>), dim3((a.Nk + 127) / 128, a.Hk, a.B), dim3(256), lds, s, a);
  if (a.far_chunks) {
    PT_ENSURE_LDS((win_bwd_kv_kernel<T, DP, true>), lds_sink);
    PT_LAUNCH((win_bwd_kv_kernel<T, DP, true>), dim3((a.sinks + 31) / 32 * a.far_chunks, a.H, a.B), dim3(256), lds_sink, s, a);
    const int64_t n = (int64_t)a.B * a.Hk * 2 * a.sinks * a.D;
    PT_LAUNCH(win_bwd_join_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a, 1 + a.far_chunks * (a.H / a.Hk) * 4);
  }
  return 0;
}

int launch_window_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int64_t* st, const int* lengths, int B, int Nq, int Nk,
                      int H, int Hk, int D, int left, int right, int sinks, float scale, int dtype, hipStream_t s) {
  if (check_win("attention_window_fwd", B, Nq, Nk, H, Hk, D, left, right, sinks, scale, dtype)) return 1;
  PT_CHECK(q && k && v && o && st, "attention_window_fwd: null argument");
  PT_CHECK(aligned16(q, st, 3, dtype) && aligned16(k, st + 3, 3, dtype) && aligned16(v, st + 6, 3, dtype) && !((uintptr_t)o & 15),
           "attention_window_fwd: addresses and strides must be multiples of 16 bytes");
  const WinArgs w = win_args(q, k, v, st, lengths, B, Nq, Nk, H, Hk, D, left, right, sinks, scale);
  WinArgs a = w;
  a.o = o; a.lse = lse;
  if (dtype) return D <= 64 ? run_win_fwd<__bf16, 64>(a, s) : run_win_fwd<__bf16, 128>(a, s);
  return D <= 64 ? run_win_fwd<float, 64>(a, s) : run_win_fwd<float, 128>(a, s);
}

size_t window_bwd_workspace(int B, int Nq, int Nk, int H, int Hk, int D, int left, int right, int sinks) {
  if (check_win("attention_window_bwd", B, Nq, Nk, H, Hk, D, left, right, sinks, 1.f, 0)) return 0;
  const int64_t st[9] = {};
  const WinArgs a = win_args(nullptr, nullptr, nullptr, st, nullptr, B, Nq, Nk, H, Hk, D, left, right, sinks, 1.f);
  const size_t delta = ((size_t)B * H * Nq * 4 + 255) / 256 * 256;
  return delta + (a.far_chunks ? (size_t)(1 + a.far_chunks * (H / Hk) * 4) * B * Hk * 2 * a.sinks * D * 4 : 0);
}

int launch_window_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse, void* dq, void* dk, void* dv,
                      const int64_t* st, const int* lengths, int B, int Nq, int Nk, int H, int Hk, int D, int left, int right, int sinks, float scale,
                      int dtype, void* ws, size_t ws_bytes, hipStream_t s) {
  if (check_win("attention_window_bwd", B, Nq, Nk, H, Hk, D, left, right, sinks, scale, dtype)) return 1;
  PT_CHECK(q && k && v && o && dout && lse && dq && dk && dv && st && ws, "attention_window_bwd: null argument");
  PT_CHECK(aligned16(q, st, 3, dtype) && aligned16(k, st + 3, 3, dtype) && aligned16(v, st + 6, 3, dtype) &&
               !(((uintptr_t)o | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)ws) & 15),
           "attention_window_bwd: addresses and strides must be multiples of 16 bytes");
  const size_t need = window_bwd_workspace(B, Nq, Nk, H, Hk, D, left, right, sinks);
  PT_CHECK(ws_bytes >= need, "attention_window_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  WinArgs a = win_args(q, k, v, st, lengths, B, Nq, Nk, H, Hk, D, left, right, sinks, scale);
  a.od = o; a.dod = dout; a.lse = const_cast<float*>(lse); a.dq = dq; a.dk = dk; a.dv = dv;
  a.delta = (float*)ws;
  a.part = a.far_chunks ? (float*)((char*)ws + ((size_t)B * H * Nq * 4 + 255) / 256 * 256) : nullptr;
  if (dtype) return D <= 64 ? run_win_bwd<__bf16, 64>(a, s) : run_win_bwd<__bf16, 128>(a, s);
  return D <= 64 ? run_win_bwd<float, 64>(a, s) : run_win_bwd<float, 128>(a, s);
}

// Slices of the visible keys: enough workgroups for every CU (four each), none with fewer than 64 keys
static int step_splits(int B, int N, int H, int Hk, int left, int sinks) {
  const int group = H / Hk, groups = (group + 7) / 8;
  const int64_t most = std::min<int64_t>(N, (int64_t)(left < 0 ? N : left) + 1 + sinks), units = (int64_t)B * Hk * groups;
  const int64_t want = ((int64_t)device_cus() * 4 + units - 1) / units;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, (most + 63) / 64), 256));
}
size_t window_step_workspace(int B, int N, int H, int Hk, int D, int left, int sinks) {
  if (check_win("attention_window_step", B, 1, N, H, Hk, D, left, 0, sinks, 1.f, 0)) return 0;
  const int n = step_splits(B, N, H, Hk, left, sinks);
  return n == 1 ? 16 : (size_t)B * H * n * (D + 2) * sizeof(float);
}

template <typename T, int L, int G>
static int run_step(const StepArgs& a, hipStream_t s) {
  const int groups = (a.H / a.Hk + G - 1) / G;
  PT_LAUNCH((win_step_kernel<T, L, G>), dim3(a.splits, a.Hk * groups, a.B), dim3(256), 0, s, a);
  if (a.splits > 1) PT_LAUNCH(win_step_join_kernel<T>, dim3((unsigned)(a.B * a.H)), dim3(128), 0, s, a);
  return 0;
}
template <typename T, int L>
static int run_step(const StepArgs& a, hipStream_t s) {
  const int group = a.H / a.Hk;
  return group == 1 ? run_step<T, L, 1>(a, s) : group == 2 ? run_step<T, L, 2>(a, s) : group <= 4 ? run_step<T, L, 4>(a, s) : run_step<T, L, 8>(a, s);
}

int launch_window_step(const void* q, const void* k, const void* v, void* o, const int64_t* st, const int* lengths, int B, int N, int H, int Hk, int D,
                       int left, int sinks, float scale, int dtype, void* ws, size_t ws_bytes, hipStream_t s) {
  if (check_win("attention_window_step", B, 1, N, H, Hk, D, left, 0, sinks, scale, dtype)) return 1;
  PT_CHECK(q && k && v && o && st && lengths && ws, "attention_window_step: null argument");
  PT_CHECK(aligned16(q, st, 2, dtype) && aligned16(k, st + 2, 3, dtype) && aligned16(v, st + 5, 3, dtype) && !(((uintptr_t)o | (uintptr_t)ws) & 15),
           "attention_window_step: addresses and strides must be multiples of 16 bytes");
  const size_t need = window_step_workspace(B, N, H, Hk, D, left, sinks);
  PT_CHECK(ws_bytes >= need, "attention_window_step: workspace of %zu bytes, %zu needed", ws_bytes, need);
  StepArgs a = {};
  a.q = q; a.k = k; a.v = v; a.o = o; a.lengths = lengths;
  for (int i = 0; i < 2; ++i) a.sq[i] = st[i];
  for (int i = 0; i < 3; ++i) { a.sk[i] = st[2 + i]; a.sv[i] = st[5 + i]; }
  a.B = B; a.N = N; a.H = H; a.Hk = Hk; a.D = D; a.left = left < 0 || left > WIN_FAR ? WIN_FAR : left; a.sinks = sinks; a.sc = scale * LOG2E;
  a.splits = step_splits(B, N, H, Hk, left, sinks);
  a.part = (float*)ws;
  if (dtype) return D <= 64 ? run_step<__bf16, 8>(a, s) : run_step<__bf16, 16>(a, s);
  return D <= 64 ? run_step<float, 8>(a, s) : run_step<float, 16>(a, s);
}

}  // namespace pt
