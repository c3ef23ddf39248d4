// Attention over a window of keys and a few first ones (sinks), forward, backward and for single tokens over a cache.
//
//   row i of a sequence stands at position t = i + (Nk - Nq); key j is visible to it where
//     j <= t + right  and  (j >= t - left  or  j < sinks)  and  j < length
//   o_i = sum_j p_ij v_j,  p_i = softmax over the visible j of scale q_i.k_j;  a row that sees nothing gives 0
//   backward, with P from the kept log-sum-exp and delta_i = do_i.o_i:
//     dV = P^T dO,  dS = P (dO V^T - delta) scale,  dQ = dS K,  dK = dS^T Q      (dK, dV summed over the query heads of a group)
//
// Bound by the matrix cores (4 D flops a visible pair forward, 14 D backward: S and dP are computed in both of its kernels, which
// costs 4 D and saves the atomics or the round trip of dQ; bf16 6 D and 20 D, see split) and, next to them, by the exponentials on the vector unit.
//
// Layout.  All products are 32 x 32 tiles with 16 contraction steps: bf16 one v_mfma_f32_32x32x16_bf16, fp32 eight
// v_mfma_f32_32x32x2_f32 on the same lanes (element e of a lane's eight is contraction step 8 (lane / 32) + e in both, so one code
// serves both types).  A result tile has its column in the lane and its rows in registers: element r is row
// (r & 3) + 8 (r >> 2) + 4 (lane / 32).  Scores are always taken so that what follows is the SECOND operand of the next product with
// exactly these registers (its contraction order being 4 + 4 rows per lane half): S^T = K Q^T then O^T += V^T P^T, and in the dK / dV
// kernel S = Q K^T then dV^T += dO^T P: probabilities never leave the registers, softmax statistics are one value per lane.
// The first operand of those second products is the transpose of a tile that lies row by row in LDS: bf16 reads it with the
// transposing ds_read_b64_tr_b16, fp32 with single words.  LDS rows hold 16-byte chunks in an order that is free of bank conflicts
// for both kinds of reads (Tile::swz).  Tiles come by
// LDS-DMA into two buffers: a tile is under way while the one before is worked on.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

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
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef const __attribute__((address_space(1))) void* glb_ptr_t;

constexpr float LOG2E = 1.4426950408889634f, SLACK = 8.f;

template <typename T> struct Types;
template <> struct Types<__bf16> { typedef bf16x8 frag; };
template <> struct Types<float> { typedef f32x8 frag; };

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
  signed char* rest;                                     // bf16: what o lost when it was rounded, a byte a value; or null
  float* part;                                           // shares of the first keys' gradients (see win_bwd_sink_kernel)
  int64_t sq[3], sk[3], sv[3];                           // strides of batch, row, head in values
  const int* lengths;
  int B, Nq, Nk, H, Hk, D, left, right, sinks;
  float sc, scale;                                       // scale * log2(e), scale
  int far, far_chunks, far_rows;                         // first row index that sees the first keys only as sinks, its chunks, rows of one
};

__device__ __forceinline__ int length_of(const WinArgs& a, int b) { return a.lengths ? min(max(a.lengths[b], 0), a.Nk) : a.Nk; }

// LDS image of a tile: rows of DP values, 16-byte chunks permuted within the row by swz(row), which is linear over xor and looks at the
// row's low four bits only.  So a lane's address for any operand of a tile is one base of its own, xor and plus constants.
template <typename T, int DP>
struct Tile {
  static constexpr int RB = DP * (int)sizeof(T), CPR = RB / 16, EPC = 16 / (int)sizeof(T);
  typedef typename Types<T>::frag frag;
  static __device__ __forceinline__ constexpr int swz(int row) {
    // 128-byte rows: two rows per turn of the banks, so the row's lowest bit is a half already
    if (RB == 128) return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
    // transposing reads take four rows of 64 bytes at a time: these go to the four quarters of the banks
    if (sizeof(T) == 2) return (row & 1) << 3 | ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
    // single words take rows r and r + 4, half of the banks each
    return ((row >> 2) & 1) << 3 | (row & 1) << 2 | ((row >> 1) & 1) << 1 | ((row >> 3) & 1);
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swz(row)) << 4); }
  // rows: lane base for 8 values along row `row` (16 s + 8 h of it)
  static __device__ __forceinline__ int row_base(int row, int h) { return at(row, sizeof(T) == 2 ? h : 2 * h); }
  static __device__ __forceinline__ frag row_frag(const unsigned char* m, int base, int s) {
    if constexpr (sizeof(T) == 2) return *reinterpret_cast<const bf16x8*>(m + (base ^ (s << 5)));
    else {
      const f32x4 x = *reinterpret_cast<const f32x4*>(m + (base ^ (s << 6))), y = *reinterpret_cast<const f32x4*>(m + (base ^ (s << 6) ^ 16));
      const frag f = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      return f;
    }
  }
  // columns: lane base for 8 values down column 32 db + lane % 32: rows row0 + 8 (e >> 2) + 4 h + (e & 3), row0 a multiple of 16
  static __device__ __forceinline__ int col_base(int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int tq = (lane >> 2) & 3, tp = lane & 3, tg = (lane >> 4) & 1;
      return at(4 * h + tq, tg * 2 + (tp >> 1)) + (tp & 1) * 8;
    } else {
      const int d = lane & 31;
      return at(4 * h, d / 4) + (d & 3) * 4;
    }
  }
};

// The column operands of 32 rows of a tile, all columns: f[s2][db] are rows OFF / RB + 16 s2 .. + 15.
// bf16: the transposing reads are asm with their wait: the compiler takes the builtin for one that may read what LDS-DMA is still
// writing and waits for every load in flight, which are the next tile's.  The caller's barriers order them.
template <typename T, int DP> struct Cols;
template <int DP>
struct Cols<__bf16, DP> {
  typedef Tile<__bf16, DP> tile;
  static constexpr int RB = tile::RB, ND = DP / 32;
  unsigned x[ND], y[ND];
  __device__ __forceinline__ Cols(const unsigned char* m, int base) {
    const unsigned at = (unsigned)(size_t)(__attribute__((address_space(3))) const unsigned char*)m + base;
#pragma unroll
    for (int db = 0; db < ND; ++db) {
      x[db] = at ^ (db << 6);
      y[db] = x[db] ^ (tile::swz(8) << 4);
    }
  }
  // columns 64 HALF .. 64 HALF + 63
  template <int OFF, int HALF>
  __device__ __forceinline__ void read_half(bf16x8 (&f)[2][2]) const {
    s16x4 r[4][2];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %2, %10 offset:%13\n\t"
        "ds_read_b64_tr_b16 %1, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %11 offset:%13\n\t"
        "ds_read_b64_tr_b16 %4, %8 offset:%14\n\tds_read_b64_tr_b16 %6, %10 offset:%15\n\t"
        "ds_read_b64_tr_b16 %5, %9 offset:%14\n\tds_read_b64_tr_b16 %7, %11 offset:%15\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[2][0]), "=&v"(r[2][1]), "=&v"(r[3][0]), "=&v"(r[3][1])
        : "v"(x[2 * HALF]), "v"(x[2 * HALF + 1]), "v"(y[2 * HALF]), "v"(y[2 * HALF + 1]), "i"(OFF), "i"(OFF + 8 * RB), "i"(OFF + 16 * RB), "i"(OFF + 24 * RB));
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        const s16x4 p = r[2 * s2][db], q = r[2 * s2 + 1][db];
        const s16x8 v = {p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
        f[s2][db] = __builtin_bit_cast(bf16x8, v);
      }
  }
  template <int OFF>
  __device__ __forceinline__ void read(bf16x8 (&f)[2][ND]) const {
    if constexpr (ND == 2) {
      read_half<OFF, 0>(f);
    } else {
      static_assert(ND == 4, "64 or 128 columns");
      s16x4 r[4][ND];
      asm volatile(
          "ds_read_b64_tr_b16 %0, %16 offset:%24\n\tds_read_b64_tr_b16 %4, %20 offset:%25\n\t"
          "ds_read_b64_tr_b16 %1, %17 offset:%24\n\tds_read_b64_tr_b16 %5, %21 offset:%25\n\t"
          "ds_read_b64_tr_b16 %2, %18 offset:%24\n\tds_read_b64_tr_b16 %6, %22 offset:%25\n\t"
          "ds_read_b64_tr_b16 %3, %19 offset:%24\n\tds_read_b64_tr_b16 %7, %23 offset:%25\n\t"
          "ds_read_b64_tr_b16 %8, %16 offset:%26\n\tds_read_b64_tr_b16 %12, %20 offset:%27\n\t"
          "ds_read_b64_tr_b16 %9, %17 offset:%26\n\tds_read_b64_tr_b16 %13, %21 offset:%27\n\t"
          "ds_read_b64_tr_b16 %10, %18 offset:%26\n\tds_read_b64_tr_b16 %14, %22 offset:%27\n\t"
          "ds_read_b64_tr_b16 %11, %19 offset:%26\n\tds_read_b64_tr_b16 %15, %23 offset:%27\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[0][2]), "=&v"(r[0][3]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[1][2]), "=&v"(r[1][3]),
            "=&v"(r[2][0]), "=&v"(r[2][1]), "=&v"(r[2][2]), "=&v"(r[2][3]), "=&v"(r[3][0]), "=&v"(r[3][1]), "=&v"(r[3][2]), "=&v"(r[3][3])
          : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(y[0]), "v"(y[1]), "v"(y[2]), "v"(y[3]), "i"(OFF), "i"(OFF + 8 * RB), "i"(OFF + 16 * RB),
            "i"(OFF + 24 * RB));
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int db = 0; db < ND; ++db) {
          const s16x4 p = r[2 * s2][db], q = r[2 * s2 + 1][db];
          const s16x8 v = {p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
          f[s2][db] = __builtin_bit_cast(bf16x8, v);
        }
    }
  }
};
template <int DP>
struct Cols<float, DP> {
  typedef Tile<float, DP> tile;
  static constexpr int RB = tile::RB, ND = DP / 32;
  const unsigned char* m;
  int base;
  __device__ __forceinline__ Cols(const unsigned char* m_, int base_) : m(m_), base(base_) {}
  template <int OFF>
  __device__ __forceinline__ void read(f32x8 (&f)[2][ND]) const {
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int db = 0; db < ND; ++db)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int r = 8 * (e >> 2) + (e & 3);
          f[s2][db][e] = *reinterpret_cast<const float*>(m + OFF + (16 * s2 + r) * RB + (base ^ (tile::swz(r) << 4) ^ (db << 7)));
        }
  }
};
// The registers of a score tile as the second operand of a product.  bf16: as the sum of two bf16 values, 2^-17 off.  One alone is 2^-8 off, and so is
// the result, however many keys share a row's weight: 1.44 times the error of rounding the exact result, and more where few rows add up.
// 8192 rows, 1028 keys, 16 heads over 4, D = 128, one value and two: forward 106 and 133 us, dQ 155 and 189, dK / dV 169 and 230
template <typename T>
__device__ __forceinline__ void split(const f32x16& p, int s2, typename Types<T>::frag& hi, typename Types<T>::frag& lo) {
#pragma unroll
  for (int e = 0; e < 8; ++e) hi[e] = (T)p[8 * s2 + e];
  if constexpr (sizeof(T) == 2)
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = (T)(p[8 * s2 + e] - (float)hi[e]);
}
// acc[db] += (columns of 32 rows)^T . p, p the registers of a score tile over these rows
template <typename T, int DP>
__device__ __forceinline__ void add_product(f32x16 (&acc)[DP / 32], const typename Types<T>::frag (&f)[2][DP / 32], const f32x16& p) {
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2) {
    typename Types<T>::frag hi, lo;
    split<T>(p, s2, hi, lo);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) acc[db] = mma(f[s2][db], hi, acc[db]);
    if constexpr (sizeof(T) == 2)
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) acc[db] = mma(f[s2][db], lo, acc[db]);
  }
}
// The same with the columns read 64 at a time, for a kernel that has no registers for all of them (dK / dV at D = 128: a tenth less)
template <int DP>
__device__ __forceinline__ void add_columns(f32x16 (&acc)[DP / 32], const Cols<__bf16, DP>& c, const f32x16& p) {
  bf16x8 hi[2], lo[2];
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2) split<__bf16>(p, s2, hi[s2], lo[s2]);
  auto half = [&](auto h) {
    constexpr int H = decltype(h)::value;
    bf16x8 f[2][2];
    c.template read_half<0, H>(f);
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
#pragma unroll
      for (int d = 0; d < 2; ++d) acc[2 * H + d] = mma(f[s2][d], hi[s2], acc[2 * H + d]);
#pragma unroll
      for (int d = 0; d < 2; ++d) acc[2 * H + d] = mma(f[s2][d], lo[s2], acc[2 * H + d]);
    }
  };
  half(std::integral_constant<int, 0>{});
  if constexpr (DP > 64) half(std::integral_constant<int, 1>{});
}
// What a value lost when it was rounded to bf16, in steps of its 24-bit pattern (-128 to 128, of which 128 is taken for 127), and the value
// that both stand for, off by a step and a half of 2^-15 at most
__device__ __forceinline__ int rest_of(float x, __bf16 r) {
  const int d = (int)(__builtin_bit_cast(unsigned, x) - ((unsigned)__builtin_bit_cast(unsigned short, r) << 16));
  return min((d + 0x80) >> 8, 127);
}
__device__ __forceinline__ float with_rest(__bf16 r, int rest) {
  return __builtin_bit_cast(float, ((unsigned)__builtin_bit_cast(unsigned short, r) << 16) + (unsigned)(rest * 256));
}

// R rows of a tile straight from memory to LDS (LDS-DMA: no registers, nothing for the compiler to wait for), by TH threads.  A wave
// writes 1 KB at a time, lane after lane, so the order of the chunks is made by the addresses that the lanes read from.  Rows behind
// the last one are that row again and columns behind D the row's first ones: such scores are masked or meet zeros of the other
// operand, and what such columns give is not stored.
template <typename T, int DP, int R, int TH>
struct Dma {
  typedef Tile<T, DP> tile;
  static constexpr int RB = tile::RB, W = TH / 64, ROWS = W * 1024 / RB, N = R / ROWS;     // rows per turn of all waves, turns
  static_assert(N >= 1 && R % ROWS == 0, "tile too small for the workgroup");
  int row, col[2];                                       // row and first byte of this lane in the first turn (and in odd turns of 8 rows)
  unsigned off[2];
  int64_t stride;                                        // bytes of a row
  __device__ __forceinline__ Dma(int D, int64_t stride_, int thread = threadIdx.x) : stride(stride_ * (int64_t)sizeof(T)) {
    const int byte = thread % TH * 16;
    row = byte / RB;
    const int chunk = (byte % RB / 16) ^ tile::swz(row), odd = chunk ^ tile::swz(ROWS);
    col[0] = chunk * tile::EPC < D ? chunk * 16 : 0;
    col[1] = odd * tile::EPC < D ? odd * 16 : 0;
    off[0] = (unsigned)(row * (int)stride + col[0]);
    off[1] = (unsigned)(row * (int)stride + col[1]);
  }
  // rows row0 .. row0 + R - 1 of base, row0 < limit
  __device__ __forceinline__ void operator()(const T* __restrict__ base, int row0, int limit, unsigned char* m) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x % TH >> 6), last = limit - 1 - row0;
    const char* from = reinterpret_cast<const char*>(base) + row0 * stride;
    if (R - 1 <= last) {                                 // a whole tile: uniform address, a lane's offset that stays the same
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const unsigned o = off[ROWS % 16 ? i & 1 : 0];
        __builtin_amdgcn_global_load_lds((glb_ptr_t)(from + i * ROWS * stride + o), (lds_ptr_t)(m + (i * W + wave) * 1024), 16, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        __builtin_amdgcn_global_load_lds((glb_ptr_t)(from + (min(row + i * ROWS, last) * (int)stride + col[ROWS % 16 ? i & 1 : 0])),
                                         (lds_ptr_t)(m + (i * W + wave) * 1024), 16, 0, 0);
      asm volatile("");                                  // keeps the two apart: merged, every tile pays for the last one's arithmetic
    }
  }
};
// The order of a block of products with their operands from LDS: P reads ahead, then R reads with each M products.  Left to itself the
// compiler reads an operand, waits for it, multiplies, and reads the next.
template <int P, int R, int M, int PRODUCTS>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, P, 0);
#pragma unroll
  for (int i = 0; i < PRODUCTS / M; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
  }
}
// loads to LDS of this wave have arrived; the barrier behind it says so of all waves
__device__ __forceinline__ void dma_wait() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// 8 values of row `row` from memory, as an operand
template <typename T>
__device__ __forceinline__ typename Types<T>::frag global_frag(const T* __restrict__ base, int64_t stride, int row, int limit, int c, int D) {
  typename Types<T>::frag f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (T)0.f;
  if (row < limit && c < D) f = *reinterpret_cast<const typename Types<T>::frag*>(base + row * stride + c);
  return f;
}
// a transposed result (lane: row `row` of the output, registers: columns) times x.  bf16: the two lanes of a row swap, so that each has
// eight neighbours to store
template <typename T, int DP>
__device__ __forceinline__ void store_transposed(T* __restrict__ base, const f32x16 (&acc)[DP / 32], int h, int D, float x, signed char* rest = nullptr) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = db * 32 + 8 * g + 4 * h;
        const f32x4 o = {acc[db][4 * g] * x, acc[db][4 * g + 1] * x, acc[db][4 * g + 2] * x, acc[db][4 * g + 3] * x};
        if (c < D) *reinterpret_cast<f32x4*>(base + c) = o;
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        unsigned w[2][2], r[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          bf16x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = acc[db][4 * (g + k) + e] * x;
            o[e] = (__bf16)y;
            r[k] |= (unsigned)(rest_of(y, o[e]) & 255) << 8 * e;
          }
          const uint2 u = __builtin_bit_cast(uint2, o);
          w[k][0] = u.x; w[k][1] = u.y;
        }
        const auto s0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false), s1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        const int c = db * 32 + 8 * (g + h);
        const u32x4 o = {s0[0], s1[0], s0[1], s1[1]};
        if (c < D) *reinterpret_cast<u32x4*>(base + c) = o;
        if (rest) {
          const auto s = __builtin_amdgcn_permlane32_swap(r[0], r[1], false, false);
          const uint2 y = {s[0], s[1]};
          if (c < D) *reinterpret_cast<uint2*>(rest + c) = y;
        }
      }
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
// Scores of invisible pairs to -infinity: keys along the registers of a transposed tile (KEYS) or along the lanes
template <bool KEYS>
__device__ __forceinline__ void mask_tile(const WinArgs& a, int len, int t, int key, int h, f32x16& st, int last = 0x7FFFFFFF) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int step = (r & 3) + 8 * (r >> 2) + 4 * h, tt = KEYS ? t : t + step, j = KEYS ? key + step : key;
    const bool on = (j <= tt + a.right) & ((j >= tt - a.left) | (j < a.sinks)) & (j < len) & (KEYS | (tt <= last));
    st[r] = on ? st[r] : -INFINITY;
  }
}
// Workgroups go to the 8 XCDs in turn, each with an L2 of its own: XCD x gets a run of neighbours in the order of the work, so that
// workgroups that read the same keys (or rows) share an L2.  Key heads of a sequence (units of `per` neighbours) go to the XCDs in turn where
// they share out evenly: sequences of a padded batch differ in length
__device__ __forceinline__ int work_item(int id, int total, int per) {
  const int x = id % 8, n = id / 8;
  if (total / per % 8 == 0) return (n / per * 8 + x) * per + n % per;
  const int q = total / 8, r = total % 8;
  return x * q + min(x, r) + n;
}
struct Place { int tile, head, kvh, b; };
// order of the work: query heads of a group, tiles, key heads, sequences
__device__ __forceinline__ Place place(const WinArgs& a, int tiles) {
  const int group = a.H / a.Hk;
  int n = work_item(blockIdx.x, gridDim.x, group * tiles);
  Place p;
  const int g = n % group; n /= group;
  p.tile = n % tiles; n /= tiles;
  p.kvh = n % a.Hk;
  p.b = n / a.Hk;
  p.head = p.kvh * group + g;
  return p;
}
// A transposed result on its way from one wave to another through LDS: `to` is the column's row of DP + 4 words there
template <int DP>
__device__ __forceinline__ void hand_over(const f32x16 (&x)[DP / 32], float* to, int h) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(to + db * 32 + 8 * g + 4 * h) = f32x4{x[db][4 * g], x[db][4 * g + 1], x[db][4 * g + 2], x[db][4 * g + 3]};
}
template <int DP>
__device__ __forceinline__ void take_over(f32x16 (&x)[DP / 32], const float* from, int h, float mine, float other) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(from + db * 32 + 8 * g + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[db][4 * g + e] = x[db][4 * g + e] * mine + y[e] * other;
    }
}
template <typename T, int DP> constexpr int key_tile() { return sizeof(T) == 2 ? 64 : 32; }
// The row kernels (forward, dQ): RW waves of 32 rows each, and SETS of them that take every SETS-th key tile and are joined at the end.
// fp32 with D up to 64 has finer workgroups: 64 rows, two sets, two of them on a CU.  Its products take 16 times bf16's time, so a workgroup of 128 rows
// is long and the chip ends unevenly: 4 padded sequences of 1200 rows, 8 heads, 257 keys 63 -> 36 us forward, 87 -> 49 dQ; two causal
// ones of 4096 537 -> 408 forward.  (One set of 64 rows, five workgroups on a CU: 52 and 71 us.)
template <typename T, int DP>
struct RowPlan {                                         // WAVES: per SIMD
  static constexpr bool FINE = sizeof(T) == 4 && DP == 64;
  static constexpr int RW = FINE ? 2 : 4, SETS = FINE ? 2 : 1, TS = RW * 64, TH = SETS * TS, ROWS = RW * 32, WAVES = DP * (int)sizeof(T) > 256 ? 1 : 2;
};

// ---------------------------------------------------------------------------
// Forward: waves of 32 rows each over common key tiles (RowPlan).  bf16, 8192 rows that see 1028 keys, 16 heads over 4, D = 128: 133 us,
// 486 TFLOP/s of visible pairs; its products (three for the formula's two) alone would take 99 us at the rate of a large matrix product on this card, the
// rest is softmax, the window's edges and loads that they do not cover.  fp32: see RowPlan
// ---------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__((RowPlan<T, DP>::TH), (RowPlan<T, DP>::WAVES)) void win_fwd_kernel(const WinArgs a) {
  typedef RowPlan<T, DP> plan;
  constexpr int SETS = plan::SETS, ROWS = plan::ROWS;
  constexpr int KT = key_tile<T, DP>(), NB = KT / 32;
  constexpr bool BF = sizeof(T) == 2;
  typedef Tile<T, DP> tile;
  constexpr int TB = KT * tile::RB;
  extern __shared__ __attribute__((aligned(1024))) unsigned char win_lds[];      // [2][K tile | V tile]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % plan::RW, set = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / plan::RW, h = lane >> 5, col = lane & 31;
  const Place at = place(a, (a.Nq + ROWS - 1) / ROWS);
  unsigned char* win_smem = win_lds + set * 4 * TB;
  const int head = at.head, b = at.b, i00 = at.tile * ROWS;
  const int len = length_of(a, b), shift = a.Nk - a.Nq;
  const int i0 = i00 + wave * 32, row = i0 + col, t = row + shift;
  const T* __restrict__ K = (const T*)a.k + b * a.sk[0] + at.kvh * a.sk[2];
  const T* __restrict__ V = (const T*)a.v + b * a.sv[0] + at.kvh * a.sv[2];
  const T* __restrict__ Q = (const T*)a.q + b * a.sq[0] + head * a.sq[2];
  int first, from, to;
  key_tiles<KT>(a, len, i00 + shift, min(i00 + ROWS - 1, a.Nq - 1) + shift, first, from, to);
  const int tiles = first + (to - from);
  auto key_of = [&](int n) { return (n < first ? n : from + n - first) * KT; };
  const Dma<T, DP, KT, plan::TS> dma_k(a.D, a.sk[1]), dma_v(a.D, a.sv[1]);
  if (set < tiles) {
    dma_k(K, key_of(set), len, win_smem);
    dma_v(V, key_of(set), len, win_smem + TB);
  }
  typename Types<T>::frag qf[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) qf[s] = global_frag(Q, a.sq[1], row, a.Nq, 16 * s + 8 * h, a.D);
  f32x16 o[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) o[db] = zero16();
  float m = -INFINITY, l = 0.f;
  const int w0 = i0 + shift, w1 = min(i0 + 31, a.Nq - 1) + shift;        // positions of this wave
  const int rb = tile::row_base(col, h), cb = tile::col_base(lane);
  dma_wait();
  for (int turn = 0; turn * SETS < tiles; ++turn) {
    const int n = turn * SETS + set;
    const unsigned char* Ks = win_smem + (turn & 1) * 2 * TB;
    const unsigned char* Vs = Ks + TB;
    const int k0 = key_of(n), k1 = k0 + KT - 1;
    if (n + SETS < tiles) {                                                 // into the other buffer: its readers passed the last barrier
      unsigned char* next = win_smem + ((turn + 1) & 1) * 2 * TB;
      dma_k(K, key_of(n + SETS), len, next);
      dma_v(V, key_of(n + SETS), len, next + TB);
    }
    if ((SETS == 1 || n < tiles) && i0 < a.Nq && k0 <= w1 + a.right && (k1 >= w0 - a.left || k0 < a.sinks)) {
      f32x16 st[NB];
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        st[x] = zero16();
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) st[x] = mma(tile::row_frag(Ks + 32 * x * tile::RB, rb, s), qf[s], st[x]);
      }
      if constexpr (BF) reads_ahead<6, 1, 1, NB * DP / 16>(); else reads_ahead<4, 2, 8, NB * DP / 2>();
      // bf16: the values' columns are on their way while the matrix cores finish the scores
      typename Types<T>::frag vf[NB][2][DP / 32];
      const Cols<T, DP> vc(Vs, cb);
      if constexpr (BF) {
        vc.template read<0>(vf[0]);
        vc.template read<32 * tile::RB>(vf[1]);
      } else {
        vc.template read<0>(vf[0]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (!(k1 <= w0 + a.right && k1 < len && (k0 >= w1 - a.left || k1 < a.sinks)))
#pragma unroll
        for (int x = 0; x < NB; ++x) mask_tile<true>(a, len, t, k0 + 32 * x, h, st[x]);
      float mx = st[0][0];
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[x][r]);
      mx = fmaxf(mx, half_other(mx)) * a.sc;
      // The base of the exponentials follows the maximum only where that has grown by 8 (or is the first one): the sums stay below
      // 2^8 times what they would be, far from fp32's range, and the results need no factor in most tiles
      if (__ballot(mx > m + SLACK)) {
        const float mn = mx > m + SLACK ? mx : m, alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
        m = mn;
        l *= alpha;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      }
      const float base = m == -INFINITY ? 0.f : m;                       // nothing visible so far: every exponential is 0
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          st[x][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[x][r], a.sc, -base));
          l += st[x][r];                                                 // this lane's half of the column; joined at the end
        }
      if constexpr (!BF && NB > 1) {
        vc.template read<32 * tile::RB>(vf[1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      add_product<T, DP>(o, vf[0], st[0]);
      if constexpr (NB > 1) add_product<T, DP>(o, vf[1], st[1]);
    }
    dma_wait();
  }
  if constexpr (SETS > 1) {                              // the other sets' sums and maxima to the first (behind the last barrier the tiles are free)
    constexpr int JW = DP + 4;
    float* rows = reinterpret_cast<float*>(win_lds) + (wave * 32 + col) * JW;
    if (set) {
      float* mine = rows + (set - 1) * ROWS * JW;
      hand_over<DP>(o, mine, h);
      if (h == 0) mine[DP] = m;
      mine[DP + 1 + h] = l;
    }
    __syncthreads();
    if (set) return;
#pragma unroll
    for (int x = 0; x < SETS - 1; ++x) {
      const float* other = rows + x * ROWS * JW;
      const float m2 = other[DP], top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
      const float f = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
      m = top;
      l = l * f + other[DP + 1 + h] * f2;
      take_over<DP>(o, other, h, f, f2);
    }
  }
  if (row >= a.Nq) return;
  l += half_other(l);
  const int64_t out = (((int64_t)b * a.Nq + row) * a.H + head) * a.D;
  store_transposed<T, DP>((T*)a.o + out, o, h, a.D, l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l), a.rest ? a.rest + out : nullptr);
  if (a.lse && h == 0) a.lse[((int64_t)b * a.H + head) * a.Nq + row] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// ---------------------------------------------------------------------------
// Backward, dQ (and delta): rows and key tiles as forward.  The case above: 189 us for four products of the formula's three (513 TFLOP/s of visible pairs)
// ---------------------------------------------------------------------------
template <typename T, int DP> constexpr int key_tile_q() { return sizeof(T) * DP <= 128 ? 64 : 32; }   // 256 registers hold no more
template <typename T, int DP>
__global__ __launch_bounds__((RowPlan<T, DP>::TH), (RowPlan<T, DP>::WAVES)) void win_bwd_q_kernel(const WinArgs a) {
  typedef RowPlan<T, DP> plan;
  constexpr int SETS = plan::SETS, ROWS = plan::ROWS;
  constexpr int KT = key_tile_q<T, DP>(), NB = KT / 32;
  constexpr bool BF = sizeof(T) == 2;
  typedef Tile<T, DP> tile;
  constexpr int TB = KT * tile::RB;
  extern __shared__ __attribute__((aligned(1024))) unsigned char win_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % plan::RW, set = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / plan::RW, h = lane >> 5, col = lane & 31;
  const Place at = place(a, (a.Nq + ROWS - 1) / ROWS);
  unsigned char* win_smem = win_lds + set * 4 * TB;
  const int head = at.head, b = at.b, i00 = at.tile * ROWS;
  const int len = length_of(a, b), shift = a.Nk - a.Nq;
  const int i0 = i00 + wave * 32, row = i0 + col, t = row + shift;
  const T* __restrict__ K = (const T*)a.k + b * a.sk[0] + at.kvh * a.sk[2];
  const T* __restrict__ V = (const T*)a.v + b * a.sv[0] + at.kvh * a.sv[2];
  const T* __restrict__ Q = (const T*)a.q + b * a.sq[0] + head * a.sq[2];
  const int64_t so = (int64_t)a.H * a.D, ob = ((int64_t)b * a.Nq * a.H + head) * a.D;
  int first, from, to;
  key_tiles<KT>(a, len, i00 + shift, min(i00 + ROWS - 1, a.Nq - 1) + shift, first, from, to);
  const int tiles = first + (to - from);
  auto key_of = [&](int n) { return (n < first ? n : from + n - first) * KT; };
  const Dma<T, DP, KT, plan::TS> dma_k(a.D, a.sk[1]), dma_v(a.D, a.sv[1]);
  if (set < tiles) {
    dma_k(K, key_of(set), len, win_smem);
    dma_v(V, key_of(set), len, win_smem + TB);
  }
  typename Types<T>::frag qf[DP / 16], gf[DP / 16];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    qf[s] = global_frag(Q, a.sq[1], row, a.Nq, 16 * s + 8 * h, a.D);
    gf[s] = global_frag((const T*)a.dod + ob, so, row, a.Nq, 16 * s + 8 * h, a.D);
    const auto of = global_frag((const T*)a.od + ob, so, row, a.Nq, 16 * s + 8 * h, a.D);
    if constexpr (BF)
      if (row < a.Nq && 16 * s + 8 * h < a.D) {
        const uint2 w = *reinterpret_cast<const uint2*>(a.rest + ob + row * so + 16 * s + 8 * h);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta += (float)gf[s][e] * with_rest(of[e], (signed char)((e < 4 ? w.x : w.y) >> 8 * (e & 3)));
        continue;
      }
#pragma unroll
    for (int e = 0; e < 8; ++e) delta += (float)gf[s][e] * (float)of[e];
  }
  delta += half_other(delta);
  const int64_t li = ((int64_t)b * a.H + head) * a.Nq + row;
  float lse = row < a.Nq ? a.lse[li] : INFINITY;
  if (row < a.Nq && h == 0 && set == 0) a.delta[li] = delta;
  asm volatile("" : "+v"(lse), "+v"(delta));             // here, not in the loop, where the wait for them would be one for the tiles too
  f32x16 dq[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) dq[db] = zero16();
  const int w0 = i0 + shift, w1 = min(i0 + 31, a.Nq - 1) + shift;
  const int rb = tile::row_base(col, h), cb = tile::col_base(lane);
  dma_wait();
  for (int turn = 0; turn * SETS < tiles; ++turn) {
    const int n = turn * SETS + set;
    const unsigned char* Ks = win_smem + (turn & 1) * 2 * TB;
    const unsigned char* Vs = Ks + TB;
    const int k0 = key_of(n), k1 = k0 + KT - 1;
    if (n + SETS < tiles) {                                                 // into the other buffer: its readers passed the last barrier
      unsigned char* next = win_smem + ((turn + 1) & 1) * 2 * TB;
      dma_k(K, key_of(n + SETS), len, next);
      dma_v(V, key_of(n + SETS), len, next + TB);
    }
    if ((SETS == 1 || n < tiles) && i0 < a.Nq && k0 <= w1 + a.right && (k1 >= w0 - a.left || k0 < a.sinks)) {
      const bool all = k1 <= w0 + a.right && k1 < len && (k0 >= w1 - a.left || k1 < a.sinks);
      f32x16 st[NB], dp[NB];
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        st[x] = zero16();
        dp[x] = zero16();
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
          st[x] = mma(tile::row_frag(Ks + 32 * x * tile::RB, rb, s), qf[s], st[x]);
          dp[x] = mma(tile::row_frag(Vs + 32 * x * tile::RB, rb, s), gf[s], dp[x]);
        }
      }
      if constexpr (BF) reads_ahead<6, 1, 1, NB * DP / 8>(); else reads_ahead<4, 2, 8, NB * DP>();
      typename Types<T>::frag kf[NB][2][DP / 32];
      const Cols<T, DP> kc(Ks, cb);
      if constexpr (BF) {
        kc.template read<0>(kf[0]);
        if constexpr (NB > 1) kc.template read<32 * tile::RB>(kf[NB - 1]);
      } else {
        kc.template read<0>(kf[0]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (!all)
#pragma unroll
        for (int x = 0; x < NB; ++x) mask_tile<true>(a, len, t, k0 + 32 * x, h, st[x]);
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          st[x][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[x][r], a.sc, -lse)) * (dp[x][r] - delta);
      add_product<T, DP>(dq, kf[0], st[0]);
      if constexpr (NB > 1) {
        if constexpr (!BF) kc.template read<32 * tile::RB>(kf[NB - 1]);
        add_product<T, DP>(dq, kf[NB - 1], st[NB - 1]);
      }
    }
    dma_wait();
  }
  if constexpr (SETS > 1) {
    float* rows = reinterpret_cast<float*>(win_lds) + (wave * 32 + col) * (DP + 4);
    if (set) hand_over<DP>(dq, rows + (set - 1) * ROWS * (DP + 4), h);
    __syncthreads();
    if (set) return;
#pragma unroll
    for (int x = 0; x < SETS - 1; ++x) take_over<DP>(dq, rows + x * ROWS * (DP + 4), h, 1.f, 1.f);
  }
  if (row < a.Nq) store_transposed<T, DP>((T*)a.dq + (((int64_t)b * a.Nq + row) * a.H + head) * a.D, dq, h, a.D, a.scale);
}

// ---------------------------------------------------------------------------
// Backward, dK and dV: 8 waves over tiles of 64 rows, all query heads of the group in turn: 4 blocks of 32 keys, for each one wave
// on the tile's first 32 rows and one on the others, added up at the end (there are too few blocks of keys to fill the chip with
// 4 waves each).  The keys stay in registers as operands; in bf16, rows of more than 128 bytes leave no room for the values beside them (two
// waves a SIMD have 256 registers each, half of them hold the results), so these are read from LDS, where they stay too.
// The case above: 230 us for six products of the formula's four (562 TFLOP/s of visible pairs).  fp32 with D up to 64: 2 blocks of keys, values in registers, two
// workgroups on a CU (105 -> 57 us where the row kernels gain as RowPlan says).
// SINK: the rows far behind the window, which see the first 32-key blocks as sinks only.  There are as many of these rows as the
// sequence is long and only a few keys, so the waves take the SAME keys and 32 rows of a tile each, the rows are cut into
// chunks, and every workgroup leaves its share in fp32; win_bwd_join_kernel adds the shares in order.
// ---------------------------------------------------------------------------
template <typename T, int DP, bool SINK>
struct KvPlan {
  static constexpr int RB = Tile<T, DP>::RB;
  static constexpr int SETS = SINK || RB > 256 ? 1 : 2;                  // waves per block of keys; 512-byte rows need a SIMD's registers for one
  static constexpr bool FINE = !SINK && RB == 256 && sizeof(T) == 4;     // fp32, D up to 64: see RowPlan
  static constexpr int BLOCKS = FINE ? 2 : 4;                            // of 32 keys (SINK: waves on one)
  static constexpr int TH = 64 * BLOCKS * SETS, QT = SINK ? (RB > 256 ? 64 : 128) : 32 * SETS, TB = QT * RB, LB = (QT < 64 ? 64 : QT) * 4;
  static constexpr bool V_LDS = RB > 128 && !FINE;
  static constexpr int KEYS = SINK ? 32 : 32 * BLOCKS;
  static constexpr int VB = V_LDS ? KEYS * RB : 0;
  static constexpr int ONE = 2 * TB + 2 * LB;                            // Q tile | dO tile | lse | delta
  static constexpr int BUF = SINK ? 1 : 2;
  static constexpr int JOIN = (SINK ? 2 : BLOCKS) * 32 * (DP + 4) * 4;        // fp32 results on their way from wave to wave
  static constexpr int LDS = VB + BUF * ONE > JOIN ? VB + BUF * ONE : JOIN;
  static_assert(LDS <= 160 * 1024 && BUF * ONE <= 128 * 1024, "LDS, and what LDS-DMA reaches of it");
};
template <typename T, int DP, bool SINK>
__global__ __launch_bounds__((KvPlan<T, DP, SINK>::TH), DP * (int)sizeof(T) > 256 ? 1 : 2) void win_bwd_kv_kernel(const WinArgs a) {
  typedef KvPlan<T, DP, SINK> plan;
  constexpr bool BF = sizeof(T) == 2;
  constexpr int QT = plan::QT, TB = plan::TB, ONE = plan::ONE, LB = plan::LB, SETS = plan::SETS, TH = plan::TH, BLOCKS = plan::BLOCKS, KEYS = plan::KEYS;
  typedef Tile<T, DP> tile;
  extern __shared__ __attribute__((aligned(1024))) unsigned char win_smem[];      // [BUF][ONE] | values
  unsigned char* bufs = win_smem;
  unsigned char* Vs = win_smem + plan::BUF * ONE;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
  const int group = a.H / a.Hk, shift = a.Nk - a.Nq;
  const int blocks = (a.sinks + 31) / 32;                                // of 32 first keys
  int b, kvh, kb, item, chunk = 0;                                       // kb: first key of the workgroup
  if constexpr (SINK) {
    item = blockIdx.x;
    kb = item % blocks * 32; item /= blocks;
    chunk = item % a.far_chunks; item /= a.far_chunks;
    b = item / a.H;
    item %= a.H;                                                         // the query head
    kvh = item / group;
  } else {
    const int tiles = (a.Nk + KEYS - 1) / KEYS;
    item = work_item(blockIdx.x, gridDim.x, tiles);
    kb = item % tiles * KEYS; item /= tiles;
    kvh = item % a.Hk;
    b = item / a.Hk;
  }
  const int len = length_of(a, b);
  const int k0 = SINK ? kb : kb + wave % BLOCKS * 32, key = k0 + col;
  const int sub = SINK ? wave * 32 : wave / BLOCKS * 32;                   // this wave's rows of a tile
  const T* __restrict__ K = (const T*)a.k + b * a.sk[0] + kvh * a.sk[2];
  const T* __restrict__ V = (const T*)a.v + b * a.sv[0] + kvh * a.sv[2];
  // rows that this workgroup looks at
  int r0, r1;
  if constexpr (SINK) {
    r0 = a.far + chunk * a.far_rows;
    r1 = kb >= len ? 0 : min(r0 + a.far_rows, a.Nq);                     // no such key: nothing is read, the share is zeros
  } else {
    r0 = max(kb - a.right - shift, 0) / QT * QT;
    // the other kernel takes the sinks' rows from a.far on, which is behind the window of the first 128 keys
    r1 = kb >= len ? 0 : (int)min((int64_t)(kb < a.sinks ? 127 : kb + KEYS - 1) + a.left - shift + 1, (int64_t)a.Nq);
  }
  const int per = r1 > r0 ? (r1 - r0 + QT - 1) / QT : 0, total = SINK ? per : per * group;
  const int64_t so = (int64_t)a.H * a.D;
  int fh = SINK ? item : kvh * group, fr = r0;                           // head and first row of the next tile
  auto fetch = [&](unsigned char* m) {
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));                                     // made anew for every tile, these offsets take no registers in between
    const Dma<T, DP, QT, TH> dma_q(a.D, a.sq[1], thread), dma_g(a.D, so, thread);
    dma_q((const T*)a.q + b * a.sq[0] + fh * a.sq[2], fr, a.Nq, m);
    dma_g((const T*)a.dod + ((int64_t)b * a.Nq * a.H + fh) * a.D, fr, a.Nq, m + TB);
    // lse by the first wave(s), delta by the next; rows behind the last one are masked
    if (wave < 2 * LB / 256) {
      const int part = wave % (LB / 256);
      const float* from = (wave < LB / 256 ? a.lse : a.delta) + ((int64_t)b * a.H + fh) * a.Nq;
      __builtin_amdgcn_global_load_lds((glb_ptr_t)(from + min(fr + part * 64 + (thread & 63), a.Nq - 1)), (lds_ptr_t)(m + 2 * TB + wave * 256), 4, 0, 0);
    }
    fr += QT;
    if (fr >= r1) { fr = r0; ++fh; }
  };
  if (total > 0) {
    if constexpr (!SINK) fetch(bufs);
    // through registers: LDS-DMA does not reach behind 128 KB.  Zeros behind the last key and behind D
    if constexpr (plan::V_LDS)
#pragma unroll 4
      for (int e = threadIdx.x; e < plan::KEYS * tile::CPR; e += TH) {
        const int r = e / tile::CPR, c = e % tile::CPR * tile::EPC;
        u32x4 x = {0u, 0u, 0u, 0u};
        if (kb + r < len && c < a.D) x = *reinterpret_cast<const u32x4*>(V + (kb + r) * a.sv[1] + c);
        *reinterpret_cast<u32x4*>(Vs + tile::at(r, c / tile::EPC)) = x;
      }
  }
  typename Types<T>::frag kf[DP / 16], vf[plan::V_LDS ? 1 : DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    kf[s] = global_frag(K, a.sk[1], key, len, 16 * s + 8 * h, a.D);
    if constexpr (!plan::V_LDS) vf[s] = global_frag(V, a.sv[1], key, len, 16 * s + 8 * h, a.D);
  }
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) { dk[db] = zero16(); dv[db] = zero16(); }
  const int rb = tile::row_base(col, h), cb = tile::col_base(lane);
  const unsigned char* Vw = Vs + (SINK ? 0 : wave % BLOCKS * 32 * tile::RB);
  if constexpr (!SINK) dma_wait();
  int cr = r0;                                                           // first row of the current tile
  for (int n = 0; n < total; ++n) {
    if constexpr (SINK) {                                                // few tiles: one buffer, and two workgroups on a CU
      fetch(bufs);
      dma_wait();
    }
    const int t0 = cr + sub + shift, t1 = t0 + 31;
    cr = cr + QT >= r1 ? r0 : cr + QT;
    const unsigned char* Qs = bufs + (SINK ? 0 : (n & 1) * ONE) + sub * tile::RB;
    const unsigned char* Gs = Qs + TB;
    const float* ls = reinterpret_cast<const float*>(bufs + (SINK ? 0 : (n & 1) * ONE) + 2 * TB) + sub;
    if (!SINK && n + 1 < total) fetch(bufs + ((n + 1) & 1) * ONE);
    if (sub < QT && k0 <= t1 + a.right && (k0 + 31 >= t0 - a.left || k0 < a.sinks) && k0 < len) {
      const bool all = k0 + 31 <= t0 + a.right && k0 + 31 < len && (k0 >= t1 - a.left || k0 + 31 < a.sinks) && t1 - shift < r1;
      int rl = rb, cl = cb;                                              // made here, the addresses of a block's operands do not take the registers of all blocks
      asm volatile("" : "+v"(rl), "+v"(cl));
      f32x16 st = zero16(), dp = zero16();
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        st = mma(tile::row_frag(Qs, rl, s), kf[s], st);
        if constexpr (plan::V_LDS) dp = mma(tile::row_frag(Gs, rl, s), tile::row_frag(Vw, rl, s), dp);
        else dp = mma(tile::row_frag(Gs, rl, s), vf[s], dp);
      }
      constexpr int READS = plan::V_LDS ? 3 : 2;                         // for two products
      if constexpr (BF) reads_ahead<2 * READS, READS, 2, DP / 8>(); else reads_ahead<2 * READS, READS * 2, 16, DP>();
      typename Types<T>::frag f[2][DP / 32];
      if constexpr (!BF) {
        Cols<T, DP>(Gs, cl).template read<0>(f);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (!all) mask_tile<false>(a, len, t0, key, h, st, r1 - 1 + shift);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 L4 = *reinterpret_cast<const f32x4*>(ls + 8 * g + 4 * h), D4 = *reinterpret_cast<const f32x4*>(ls + LB / 4 + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          st[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], a.sc, -L4[e]));
          dp[r] = st[r] * (dp[r] - D4[e]);
        }
      }
      if constexpr (BF) {
        add_columns<DP>(dv, Cols<T, DP>(Gs, cl), st);
        add_columns<DP>(dk, Cols<T, DP>(Qs, cl), dp);
      } else if constexpr (plan::V_LDS) {
        typename Types<T>::frag f2[2][DP / 32];
        Cols<T, DP>(Qs, cl).template read<0>(f2);
        __builtin_amdgcn_sched_barrier(0);
        add_product<T, DP>(dv, f, st);
        add_product<T, DP>(dk, f2, dp);
      } else {
        add_product<T, DP>(dv, f, st);
        Cols<T, DP>(Qs, cl).template read<0>(f);
        add_product<T, DP>(dk, f, dp);
      }
    }
    if constexpr (SINK) __syncthreads();
    else dma_wait();
  }
  // the waves of one block of keys, one after the other (behind the last barrier the tiles are free)
  float* join = reinterpret_cast<float*>(win_smem);
  constexpr int JW = DP + 4;                                             // words of a key's row: 16-byte pieces of 32 rows on different banks
  auto pass = [&](f32x16 (&x)[DP / 32], float* m, bool put) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4* p = reinterpret_cast<f32x4*>(m + col * JW + db * 32 + 8 * g + 4 * h);
        if (put) *p = f32x4{x[db][4 * g], x[db][4 * g + 1], x[db][4 * g + 2], x[db][4 * g + 3]};
        else {
          const f32x4 y = *p;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[db][4 * g + e] += y[e];
        }
      }
  };
  if constexpr (SINK) {
#pragma unroll 1
    for (int w = 4 * SETS - 1; w > 0; --w) {                                        // wave w hands its sums to wave w - 1
      if (wave == w) { pass(dk, join, true); pass(dv, join + 32 * JW, true); }
      __syncthreads();
      if (wave == w - 1) { pass(dk, join, false); pass(dv, join + 32 * JW, false); }
      __syncthreads();
    }
    if (wave || key >= a.sinks) return;
    // share [slot][b][kvh][2][sinks][D]; slot 0 is the window's part
    const int slot = 1 + chunk * group + item % group;
    float* out = a.part + ((((int64_t)slot * a.B + b) * a.Hk + kvh) * 2 * a.sinks + key) * a.D;
    store_transposed<float, DP>(out, dk, h, a.D, a.scale);
    store_transposed<float, DP>(out + (int64_t)a.sinks * a.D, dv, h, a.D, 1.f);
  } else {
    if constexpr (SETS == 2) {
      float* mine = join + wave % BLOCKS * 32 * JW;
      if (wave >= BLOCKS) pass(dk, mine, true);
      __syncthreads();
      if (wave < BLOCKS) pass(dk, mine, false);
      __syncthreads();
      if (wave >= BLOCKS) pass(dv, mine, true);
      __syncthreads();
      if (wave >= BLOCKS) return;
      pass(dv, mine, false);
    }
    if (key >= a.Nk) return;
    if (a.part && key < a.sinks) {
      float* out = a.part + (((int64_t)b * a.Hk + kvh) * 2 * a.sinks + key) * a.D;
      store_transposed<float, DP>(out, dk, h, a.D, a.scale);
      store_transposed<float, DP>(out + (int64_t)a.sinks * a.D, dv, h, a.D, 1.f);
    } else {
      const int64_t to = (((int64_t)b * a.Nk + key) * a.Hk + kvh) * a.D;
      store_transposed<T, DP>((T*)a.dk + to, dk, h, a.D, a.scale);
      store_transposed<T, DP>((T*)a.dv + to, dv, h, a.D, 1.f);
    }
  }
}

// the first keys' gradients: 16 values a workgroup at a time, each the sum of 16 runs of the shares
template <typename T>
__global__ __launch_bounds__(256) void win_bwd_join_kernel(const WinArgs a, int slots) {
  const int64_t n = (int64_t)a.B * a.Hk * 2 * a.sinks * a.D;
  __shared__ float red[16][16];
  for (int64_t first = (int64_t)blockIdx.x * 16; first < n; first += (int64_t)gridDim.x * 16) {
    const int64_t i = first + (threadIdx.x & 15);
    float s = 0.f;
    if (i < n) {
#pragma unroll 8
      for (int k = threadIdx.x >> 4; k < slots; k += 16) s += a.part[k * n + i];
    }
    red[threadIdx.x >> 4][threadIdx.x & 15] = s;
    __syncthreads();
    if (threadIdx.x < 16 && i < n) {
      s = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) s += red[k][threadIdx.x];
      int64_t r = i;
      const int d = (int)(r % a.D); r /= a.D;
      const int key = (int)(r % a.sinks); r /= a.sinks;
      const int which = (int)(r & 1); r >>= 1;
      const int kvh = (int)(r % a.Hk), b = (int)(r / a.Hk);
      ((T*)(which ? a.dv : a.dk))[(((int64_t)b * a.Nk + key) * a.Hk + kvh) * a.D + d] = (T)s;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// One token: scores of the query heads of a group against the visible keys of its sequence.  Bound by HBM: every visible key and value
// is read once for all heads of the group.  Visible keys are cut into slices where there are few sequences, joined by a second kernel.
//
// win_step_kernel: on the vector unit straight from memory: L lanes hold a key's row (8 values each), the wave's 64 / L lane groups walk
// keys side by side, each with its own running maximum and sum, joined at the end.  fp32, and few short sequences of either type.
// win_step_group_kernel: bf16 on the matrix cores.
// Read rates over all visible keys and values: 64 sequences of some 3100 keys, 64 heads over 8, D = 128: 140 us, 6.0 TB/s (vector unit: 303);
// 32 heads over 8: 159 us for 986 MB, 6.2 TB/s (183); 8 over 8, D = 64, 393 MB: 75 us; one sequence of 18,000 keys, 74 MB: 18 us;
// fp32, 214 MB: 40 us
// ---------------------------------------------------------------------------
struct StepArgs {
  const void* q; const void* k; const void* v; void* o; const int* lengths;
  int64_t sq[2], sk[3], sv[3];                           // q: batch, head; caches: batch, row, head
  int B, N, H, Hk, D, left, sinks, splits;
  float sc;
  float* part;                                           // [B][H][splits][D + 2]: unnormalised output, maximum, sum
};

template <bool STREAM, typename F>
__device__ __forceinline__ F load_cache(const F* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}

// W waves: 16 where one workgroup takes all keys of its heads, 4 otherwise
template <typename T, int L, int G, int W, bool STREAM>
__global__ __launch_bounds__(W * 64) void win_step_kernel(const StepArgs a) {
  constexpr int KW = 64 / L, U = W == 4 || sizeof(T) == 2 ? 4 : 2;   // keys side by side in a wave, and turns whose loads go out together
  typedef typename Types<T>::frag frag;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane % L, sub = lane / L;
  const int groups = (a.H / a.Hk + G - 1) / G;
  const int split = blockIdx.x, kvh = blockIdx.y / groups, g0 = (blockIdx.y % groups) * G, b = blockIdx.z;
  const int group = a.H / a.Hk, heads = min(G, group - g0), h0 = kvh * group + g0;
  const int len = min(max(a.lengths[b], 0), a.N), t = len - 1;
  // the visible keys in order: [0, ns) sinks, then [lo, len)
  const int lo = max(t - a.left, 0), ns = min(min(a.sinks, lo), len), seen = len > 0 ? ns + (len - lo) : 0;
  const int per = (seen + a.splits - 1) / a.splits, n0 = min(split * per, seen), n1 = min(n0 + per, seen);
  const bool in = li * 8 < a.D;
  const int col = in ? li * 8 : 0;
  const T* __restrict__ K = (const T*)a.k + b * a.sk[0] + kvh * a.sk[2] + col;
  const T* __restrict__ V = (const T*)a.v + b * a.sv[0] + kvh * a.sv[2] + col;
  const frag zero = {};
  float q[G][8], acc[G][8], m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const frag f = *reinterpret_cast<const frag*>((const T*)a.q + b * a.sq[0] + (h0 + min(g, heads - 1)) * a.sq[1] + col);
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) { q[g][e] = in ? (float)f[e] * a.sc : 0.f; acc[g][e] = 0.f; }
  }
  for (int n = n0 + wave * KW * U; n < n1; n += W * KW * U) {
    frag k[U], v[U];
    // all loads first, without branches: rows behind the slice repeat its last one, columns behind D the first ones, and both
    // count as zeros, whatever they hold
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(n + u * KW + sub, n1 - 1), j = i < ns ? i : lo + i - ns;
      k[u] = load_cache<STREAM>(reinterpret_cast<const frag*>(K + j * a.sk[1]));
      v[u] = load_cache<STREAM>(reinterpret_cast<const frag*>(V + j * a.sv[1]));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = in && n + u * KW + sub < n1;
      k[u] = in ? k[u] : zero;
      v[u] = on ? v[u] : zero;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float s[U], mx = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf(q[g][e], (float)k[u][e], d);
#pragma unroll
        for (int x = 1; x < L; x <<= 1) d += __shfl_xor(d, x);
        s[u] = n + u * KW + sub < n1 ? d : -INFINITY;
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
        for (int e = 0; e < 8; ++e) acc[g][e] = fmaf(p, (float)v[u][e], acc[g][e]);
      }
    }
  }
  // join the lane groups, then the waves
  __shared__ float red[W][G][L * 8 + 2];
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
  for (int x = threadIdx.x; x < heads * L * 8; x += W * 64) {
    const int g = x / (L * 8), d = x % (L * 8);
    if (d >= a.D) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, red[w][g][L * 8]);
    const float base = top == -INFINITY ? 0.f : top;
    float s = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
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

// The same in bf16: up to 32 heads of a group are the columns of a 32 x 32 tile, 32 keys its rows, as in the forward kernel.  Columns
// without a head cost matrix time that the loads leave over: with one head in use it is as fast as the vector unit, with eight, where
// the vector unit is the bound, more than twice.  Every wave walks tiles of its own through LDS-DMA into two buffers, without
// barriers.  Probabilities enter the second product as sums of two bf16 values: the matrix cores have the time (64 sequences, 986 MB: 156.9 us
// with one, 159.1 with two), and the result is rounded once.
constexpr int STEP_WAVES = 4;
template <int DP, bool STREAM>
__global__ __launch_bounds__(STEP_WAVES * 64) void win_step_group_kernel(const StepArgs a) {
  typedef __bf16 T;
  typedef Tile<T, DP> tile;
  constexpr int RB = tile::RB, TB = 32 * RB, ROWS = 1024 / RB, N = 32 / ROWS, ND = DP / 32, W = STEP_WAVES;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const int group = a.H / a.Hk, groups = (group + 31) / 32;
  const int split = blockIdx.x, kvh = blockIdx.y / groups, g0 = (blockIdx.y % groups) * 32, b = blockIdx.z;
  const int heads = min(32, group - g0), h0 = kvh * group + g0;
  const int len = min(max(a.lengths[b], 0), a.N), t = len - 1;
  const int lo = max(t - a.left, 0), ns = min(min(a.sinks, lo), len), seen = len > 0 ? ns + (len - lo) : 0;
  const int per = ((seen + a.splits - 1) / a.splits + 31) / 32 * 32, n0 = min(split * per, seen), n1 = min(n0 + per, seen);
  const char* K = (const char*)((const T*)a.k + b * a.sk[0] + kvh * a.sk[2]);
  const char* V = (const char*)((const T*)a.v + b * a.sv[0] + kvh * a.sv[2]);
  unsigned char* m = lds + wave * 4 * TB;                // two buffers of keys and values
  const int row = lane * 16 / RB, chunk = (lane * 16 % RB / 16) ^ tile::swz(row);
  auto fetch = [&](int n, unsigned char* to) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = min(n + i * ROWS + row, n1 - 1), j = x < ns ? x : lo + x - ns, at = chunk ^ tile::swz(i * ROWS & 15);
      const int col = at * 8 < a.D ? at * 16 : 0;
      __builtin_amdgcn_global_load_lds((glb_ptr_t)(K + j * a.sk[1] * 2 + col), (lds_ptr_t)(to + i * 1024), 16, 0, STREAM ? 2 : 0);
      __builtin_amdgcn_global_load_lds((glb_ptr_t)(V + j * a.sv[1] * 2 + col), (lds_ptr_t)(to + TB + i * 1024), 16, 0, STREAM ? 2 : 0);
    }
  };
  const int first = n0 + wave * 32;
  if (first < n1) fetch(first, m);
  bf16x8 q[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) q[s] = global_frag<T>((const T*)a.q + b * a.sq[0] + h0 * a.sq[1], a.sq[1], c, heads, 16 * s + 8 * h, a.D);
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = zero16();
  float top = -INFINITY, l = 0.f;
  const int kb = tile::row_base(c, h), vb = tile::col_base(lane);
  int turn = 0;
  for (int n = first; n < n1; n += W * 32, turn ^= 1) {
    unsigned char* now = m + turn * 2 * TB;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (n + W * 32 < n1) fetch(n + W * 32, m + (turn ^ 1) * 2 * TB);
    f32x16 st = zero16();
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) st = mma(tile::row_frag(now, kb, s), q[s], st);
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      st[r] *= a.sc;
      if (n + 32 > n1) st[r] = n + (r & 3) + 8 * (r >> 2) + 4 * h < n1 ? st[r] : -INFINITY;
      mx = fmaxf(mx, st[r]);
    }
    mx = fmaxf(mx, half_other(mx));
    const float up = fmaxf(top, mx), base = up == -INFINITY ? 0.f : up, alpha = __builtin_amdgcn_exp2f(top - base);
    top = up;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] *= alpha;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      st[r] = __builtin_amdgcn_exp2f(st[r] - base);
      l += st[r];
    }
    bf16x8 f[2][ND];
    Cols<T, DP>(now + TB, vb).template read<0>(f);
    add_product<T, DP>(acc, f, st);
  }
  l += half_other(l);
  // join the waves
  float* red = (float*)lds;                              // [W][heads][DP + 4]: output, maximum, sum
  constexpr int RW = DP + 4;
  __syncthreads();
  if (c < heads) {
    float* out = red + (wave * heads + c) * RW;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 x = {acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
        *reinterpret_cast<f32x4*>(out + d * 32 + 8 * g + 4 * h) = x;
      }
    if (!h) { out[DP] = top; out[DP + 1] = l; }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < heads * DP; x += W * 64) {
    const int g = x / DP, d = x % DP;
    if (d >= a.D) continue;
    float most = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) most = fmaxf(most, red[(w * heads + g) * RW + DP]);
    const float base = most == -INFINITY ? 0.f : most;
    float s = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* in = red + (w * heads + g) * RW;
      const float f = __builtin_amdgcn_exp2f(in[DP] - base);
      s += f * in[DP + 1];
      y += f * in[d];
    }
    const int64_t oh = (int64_t)b * a.H + h0 + g;
    if (a.splits == 1) {
      ((T*)a.o)[oh * a.D + d] = (T)(s == 0.f ? 0.f : y / s);
    } else {
      float* out = a.part + (oh * a.splits + split) * (a.D + 2);
      out[d] = y;
      if (d == 0) { out[a.D] = most; out[a.D + 1] = s; }
    }
  }
}
// Joins the slices of one head: a lane takes the maximum and the sum of every 64th slice, a thread a column of every JOIN-th (8; 2 where there
// are no more than 8 slices: 512 heads of 2 slices, 3.5 us less)
constexpr int STEP_SPLITS = 256;
template <typename T, int JOIN>
__global__ __launch_bounds__(JOIN * 128) void win_step_join_kernel(const StepArgs a) {
  const int64_t oh = blockIdx.x;
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 7, col = threadIdx.x & 127, d = min(col, a.D - 1), row = a.D + 2;
  const float* p = a.part + oh * a.splits * row;
  float w[STEP_SPLITS / 64], y[64 / JOIN], l = 0.f, top = -INFINITY;
#pragma unroll
  for (int i = 0; i < STEP_SPLITS / 64; ++i) {
    w[i] = i * 64 + lane < a.splits ? p[(i * 64 + lane) * row + a.D] : -INFINITY;
    top = fmaxf(top, w[i]);
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < STEP_SPLITS / 64; ++i) {
    w[i] = __builtin_amdgcn_exp2f(w[i] - base);
    if (i * 64 + lane < a.splits) l += w[i] * p[(i * 64 + lane) * row + a.D + 1];
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < STEP_SPLITS / 64; ++i) {
    if (i * 64 >= a.splits) break;
#pragma unroll
    for (int s = 0; s < 64 / JOIN; ++s) y[s] = p[min(i * 64 + s * JOIN + part, a.splits - 1) * row + d];
#pragma unroll
    for (int s = 0; s < 64 / JOIN; ++s) {
      const float f = __shfl(w[i], s * JOIN + part);
      if (i * 64 + s * JOIN + part < a.splits) sum += f * y[s];
    }
  }
  __shared__ float red[JOIN][128];
  red[part][col] = sum;
  __syncthreads();
  if ((int)threadIdx.x >= a.D) return;
  sum = 0.f;
#pragma unroll
  for (int x = 0; x < JOIN; ++x) sum += red[x][threadIdx.x];
  ((T*)a.o)[oh * a.D + d] = (T)(l == 0.f ? 0.f : sum / l);
}

// ---------------------------------------------------------------------------
constexpr int WIN_FAR = 1 << 29, WIN_MAX = 1 << 28;

static int check_win(const char* who, int B, int Nq, int Nk, int H, int Hk, int D, int left, int right, int sinks, float scale, int dtype) {
  PT_CHECK(B >= 1 && B <= 65535 && Nq >= 1 && Nk >= Nq && Nk <= WIN_MAX, "%s: %d sequences of %d rows and %d keys", who, B, Nq, Nk);
  PT_CHECK(H >= 1 && H <= 65535 && Hk >= 1 && H % Hk == 0, "%s: %d query heads over %d key heads", who, H, Hk);
  PT_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "%s: head dimension %d (a multiple of 8 up to 128)", who, D);
  PT_CHECK((int64_t)((Nk + 127) / 128) * H * B < (1 << 28), "%s: too many rows and heads", who);
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
// a tile's rows are addressed by 32-bit offsets from its first
static bool near_rows(const int64_t* s) {
  for (int i = 0; i < 9; i += 3)
    if (s[i + 1] < 0 || s[i + 1] > (1 << 20)) return false;
  return true;
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
    const int rows = Nq - a.far, want = std::max(1, 1024 / (B * H));       // about four workgroups per CU, a tile of 256 rows each at least
    a.far_rows = std::max(256, ((rows + want - 1) / want + 255) / 256 * 256);
    a.far_chunks = (rows + a.far_rows - 1) / a.far_rows;
  }
  return a;
}

// a launch holds less than 2^32 threads
static bool one_launch(int64_t blocks, int threads) { return blocks * threads < ((int64_t)1 << 32); }
static int64_t win_blocks(const WinArgs& a, int rows) { return (int64_t)((a.Nq + rows - 1) / rows) * a.H * a.B; }

template <typename T, int DP>
static int run_win_fwd(const WinArgs& a, hipStream_t s) {
  typedef RowPlan<T, DP> plan;
  constexpr int lds = plan::SETS * 4 * key_tile<T, DP>() * Tile<T, DP>::RB;
  PT_CHECK(one_launch(win_blocks(a, plan::ROWS), plan::TH), "attention_window_fwd: too many rows and heads");
  PT_ENSURE_LDS((win_fwd_kernel<T, DP>), lds);
  PT_LAUNCH((win_fwd_kernel<T, DP>), dim3((unsigned)win_blocks(a, plan::ROWS)), dim3(plan::TH), lds, s, a);
  return 0;
}
static size_t lse_bytes(int B, int Nq, int H) { return ((size_t)B * H * Nq * 4 + 255) / 256 * 256; }
size_t window_stats_bytes(int B, int Nq, int H, int D, int dtype) {
  if (check_win("attention_window_fwd", B, Nq, Nq, H, H, D, 0, 0, 0, 1.f, dtype)) return 0;
  return lse_bytes(B, Nq, H) + (dtype ? (size_t)B * Nq * H * D : 0);
}
template <typename T, int DP>
static int run_win_bwd(const WinArgs& a, hipStream_t s) {
  typedef RowPlan<T, DP> plan;
  constexpr int lds = plan::SETS * 4 * key_tile_q<T, DP>() * Tile<T, DP>::RB, lds_kv = KvPlan<T, DP, false>::LDS, lds_sink = KvPlan<T, DP, true>::LDS;
  typedef KvPlan<T, DP, false> kv;
  const int64_t key_blocks = (int64_t)((a.Nk + kv::KEYS - 1) / kv::KEYS) * a.Hk * a.B, sink_blocks = (int64_t)((a.sinks + 31) / 32) * a.far_chunks * a.H * a.B;
  PT_CHECK(one_launch(win_blocks(a, plan::ROWS), plan::TH) && one_launch(key_blocks, kv::TH) && one_launch(sink_blocks, KvPlan<T, DP, true>::TH),
           "attention_window_bwd: too many rows and heads");
  PT_ENSURE_LDS((win_bwd_q_kernel<T, DP>), lds);
  PT_LAUNCH((win_bwd_q_kernel<T, DP>), dim3((unsigned)win_blocks(a, plan::ROWS)), dim3(plan::TH), lds, s, a);
  PT_ENSURE_LDS((win_bwd_kv_kernel<T, DP, false>), lds_kv);
  PT_LAUNCH((win_bwd_kv_kernel<T, DP, false>), dim3((unsigned)key_blocks), dim3(kv::TH), lds_kv, s, a);
  if (a.far_chunks) {
    PT_ENSURE_LDS((win_bwd_kv_kernel<T, DP, true>), lds_sink);
    PT_LAUNCH((win_bwd_kv_kernel<T, DP, true>), dim3((unsigned)sink_blocks), dim3(KvPlan<T, DP, true>::TH), lds_sink, s, a);
    const int64_t n = (int64_t)a.B * a.Hk * 2 * a.sinks * a.D;
    PT_LAUNCH(win_bwd_join_kernel<T>, dim3((unsigned)std::min<int64_t>((n + 15) / 16, 1 << 20)), dim3(256), 0, s, a, 1 + a.far_chunks * (a.H / a.Hk));
  }
  return 0;
}

int launch_window_fwd(const void* q, const void* k, const void* v, void* o, void* stats, const int64_t* st, const int* lengths, int B, int Nq, int Nk,
                      int H, int Hk, int D, int left, int right, int sinks, float scale, int dtype, hipStream_t s) {
  if (check_win("attention_window_fwd", B, Nq, Nk, H, Hk, D, left, right, sinks, scale, dtype)) return 1;
  PT_CHECK(q && k && v && o && st, "attention_window_fwd: null argument");
  PT_CHECK(aligned16(q, st, 3, dtype) && aligned16(k, st + 3, 3, dtype) && aligned16(v, st + 6, 3, dtype) && !((uintptr_t)o & 15),
           "attention_window_fwd: addresses and strides must be multiples of 16 bytes");
  PT_CHECK(near_rows(st) && (int64_t)H * D <= (1 << 20), "attention_window_fwd: rows are more than 2^20 values apart");
  PT_CHECK(!((uintptr_t)stats & 15), "attention_window_fwd: stats must be aligned to 16 bytes");
  WinArgs a = win_args(q, k, v, st, lengths, B, Nq, Nk, H, Hk, D, left, right, sinks, scale);
  a.o = o; a.lse = (float*)stats;
  a.rest = dtype && stats ? (signed char*)stats + lse_bytes(B, Nq, H) : nullptr;
  if (dtype) return D <= 64 ? run_win_fwd<__bf16, 64>(a, s) : run_win_fwd<__bf16, 128>(a, s);
  return D <= 64 ? run_win_fwd<float, 64>(a, s) : run_win_fwd<float, 128>(a, s);
}

size_t window_bwd_workspace(int B, int Nq, int Nk, int H, int Hk, int D, int left, int right, int sinks) {
  if (check_win("attention_window_bwd", B, Nq, Nk, H, Hk, D, left, right, sinks, 1.f, 0)) return 0;
  const int64_t st[9] = {};
  const WinArgs a = win_args(nullptr, nullptr, nullptr, st, nullptr, B, Nq, Nk, H, Hk, D, left, right, sinks, 1.f);
  const size_t delta = ((size_t)B * H * Nq * 4 + 255) / 256 * 256;
  return delta + (a.far_chunks ? (size_t)(1 + a.far_chunks * (H / Hk)) * B * Hk * 2 * a.sinks * D * 4 : 0);
}

int launch_window_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const void* stats, void* dq, void* dk, void* dv,
                      const int64_t* st, const int* lengths, int B, int Nq, int Nk, int H, int Hk, int D, int left, int right, int sinks, float scale,
                      int dtype, void* ws, size_t ws_bytes, hipStream_t s) {
  if (check_win("attention_window_bwd", B, Nq, Nk, H, Hk, D, left, right, sinks, scale, dtype)) return 1;
  PT_CHECK(q && k && v && o && dout && stats && dq && dk && dv && st && ws, "attention_window_bwd: null argument");
  PT_CHECK(aligned16(q, st, 3, dtype) && aligned16(k, st + 3, 3, dtype) && aligned16(v, st + 6, 3, dtype) &&
               !(((uintptr_t)o | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)stats | (uintptr_t)ws) & 15),
           "attention_window_bwd: addresses and strides must be multiples of 16 bytes");
  PT_CHECK(near_rows(st) && (int64_t)H * D <= (1 << 20), "attention_window_bwd: rows are more than 2^20 values apart");
  const size_t need = window_bwd_workspace(B, Nq, Nk, H, Hk, D, left, right, sinks);
  PT_CHECK(ws_bytes >= need, "attention_window_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  WinArgs a = win_args(q, k, v, st, lengths, B, Nq, Nk, H, Hk, D, left, right, sinks, scale);
  a.od = o; a.dod = dout; a.lse = (float*)const_cast<void*>(stats); a.dq = dq; a.dk = dk; a.dv = dv;
  if (dtype) a.rest = (signed char*)const_cast<void*>(stats) + lse_bytes(B, Nq, H);
  a.delta = (float*)ws;
  a.part = a.far_chunks ? (float*)((char*)ws + ((size_t)B * H * Nq * 4 + 255) / 256 * 256) : nullptr;
  if (dtype) return D <= 64 ? run_win_bwd<__bf16, 64>(a, s) : run_win_bwd<__bf16, 128>(a, s);
  return D <= 64 ? run_win_bwd<float, 64>(a, s) : run_win_bwd<float, 128>(a, s);
}

// How a call is cut.  whole: one workgroup of 16 waves takes all visible keys of a group's heads, and there is no second kernel: few
// units of few keys, whose time is latency (one sequence of 516 keys: 20.8 -> 15.4 us a call against nine slices and their join; four of
// 1000: 6.7 us on the GPU against 9.6).  matrix: win_step_group_kernel.  stream: loads that leave the caches alone, where the cache of
// the step will not stay there: bf16 from 64 MB on (836 MB 158 -> 140 us; 202 MB, six in turn, 51 -> 45; one alone 41 -> 42), fp32
// from the 256 MB of Infinity Cache on (214 MB, alone and resident: 40 us against 55).
struct StepPlan { bool whole, matrix, stream; int heads, splits; };
static StepPlan step_plan(int B, int N, int H, int Hk, int D, int left, int sinks, int dtype) {
  const int group = H / Hk;
  const int64_t most = std::min<int64_t>(N, (int64_t)(left < 0 ? N : left) + 1 + sinks), bytes = B * (int64_t)Hk * most * D * (dtype ? 2 : 4) * 2;
  StepPlan p = {};
  p.whole = group <= 2 && most <= 1024 && (int64_t)B * Hk <= device_cus();
  p.matrix = dtype && !p.whole;
  p.stream = bytes >= (int64_t)(p.matrix ? 64 : 256) << 20;
  p.heads = p.matrix ? 32 : group == 1 ? 1 : group == 2 ? 2 : group <= 4 ? 4 : 8;
  // slices of the visible keys: as many workgroups as are there at once (LDS, or the registers of the vector kernel), none with fewer
  // than 64 keys.  Twice as many: B = 8, 53 MB 16 -> 20 us
  const int64_t at_once = (int64_t)device_cus() * (p.matrix && D > 64 ? 1 : 2), units = (int64_t)B * Hk * ((group + p.heads - 1) / p.heads);
  const int64_t slices = std::min<int64_t>(std::min<int64_t>((at_once + units - 1) / units, (most + 63) / 64), STEP_SPLITS);
  p.splits = p.whole ? 1 : (int)std::max<int64_t>(1, slices);
  return p;
}
size_t window_step_workspace(int B, int N, int H, int Hk, int D, int left, int sinks) {
  if (check_win("attention_window_step", B, 1, N, H, Hk, D, left, 0, sinks, 1.f, 0)) return 0;
  const int n = std::max(step_plan(B, N, H, Hk, D, left, sinks, 0).splits, step_plan(B, N, H, Hk, D, left, sinks, 1).splits);
  return n == 1 ? 16 : (size_t)B * H * n * (D + 2) * sizeof(float);
}

template <typename T, int L, int G, int W>
static int run_step(const StepArgs& a, const StepPlan& p, hipStream_t s) {
  const dim3 grid(a.splits, a.Hk * ((a.H / a.Hk + G - 1) / G), a.B);
  if (p.stream) PT_LAUNCH((win_step_kernel<T, L, G, W, true>), grid, dim3(W * 64), 0, s, a);
  else PT_LAUNCH((win_step_kernel<T, L, G, W, false>), grid, dim3(W * 64), 0, s, a);
  return 0;
}
template <typename T, int L>
static int run_step(const StepArgs& a, const StepPlan& p, hipStream_t s) {
  if (p.whole) return p.heads == 1 ? run_step<T, L, 1, 16>(a, p, s) : run_step<T, L, 2, 16>(a, p, s);
  if constexpr (sizeof(T) == 4)
    return p.heads == 1 ? run_step<T, L, 1, 4>(a, p, s) : p.heads == 2 ? run_step<T, L, 2, 4>(a, p, s)
                        : p.heads == 4 ? run_step<T, L, 4, 4>(a, p, s) : run_step<T, L, 8, 4>(a, p, s);
  else return 1;
}
template <int DP>
static int run_step_group(const StepArgs& a, const StepPlan& p, hipStream_t s) {
  constexpr int lds = STEP_WAVES * 4 * 32 * Tile<__bf16, DP>::RB;
  static_assert(lds >= STEP_WAVES * 32 * (DP + 4) * 4 && lds <= 128 * 1024, "buffers that LDS-DMA reaches");
  const dim3 grid(a.splits, a.Hk * ((a.H / a.Hk + 31) / 32), a.B);
  if (p.stream) {
    PT_ENSURE_LDS((win_step_group_kernel<DP, true>), lds);
    PT_LAUNCH((win_step_group_kernel<DP, true>), grid, dim3(STEP_WAVES * 64), lds, s, a);
  } else {
    PT_ENSURE_LDS((win_step_group_kernel<DP, false>), lds);
    PT_LAUNCH((win_step_group_kernel<DP, false>), grid, dim3(STEP_WAVES * 64), lds, s, a);
  }
  return 0;
}

template <typename T, int JOIN>
static int run_step_join(const StepArgs& a, hipStream_t s) {
  PT_LAUNCH((win_step_join_kernel<T, JOIN>), dim3((unsigned)((int64_t)a.B * a.H)), dim3(JOIN * 128), 0, s, a);
  return 0;
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
  const StepPlan p = step_plan(B, N, H, Hk, D, left, sinks, dtype);
  a.splits = p.splits;
  a.part = (float*)ws;
  if (p.matrix ? (D <= 64 ? run_step_group<64>(a, p, s) : run_step_group<128>(a, p, s))
               : dtype ? (D <= 64 ? run_step<__bf16, 8>(a, p, s) : run_step<__bf16, 16>(a, p, s))
                       : (D <= 64 ? run_step<float, 8>(a, p, s) : run_step<float, 16>(a, p, s)))
    return 1;
  if (p.splits == 1) return 0;
  if (p.splits <= 8) return dtype ? run_step_join<__bf16, 2>(a, s) : run_step_join<float, 2>(a, s);
  return dtype ? run_step_join<__bf16, 8>(a, s) : run_step_join<float, 8>(a, s);
}

}  // namespace pt
