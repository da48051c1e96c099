// rr_gemm.h — the tiled matrix product of the output-head losses on gfx950.
//
// acc[m][n] = sum_k A(m, k) B(n, k) for a BM x BN tile, 16-bit operands, fp32
// accumulation on the 32x32x16 MFMA.  An operand lies in memory either with k
// contiguous (its rows are m or n) or k-major (its rows are k); in LDS the tile
// keeps the orientation it has in memory, and k-major tiles are read with the
// transposing LDS read, so no operand is ever transposed in memory.
//
// LDS holds 16-byte chunks.  A fragment read takes the same chunk column of many
// rows, whose addresses differ by a multiple of the row length, so chunk columns
// are permuted by row (an XOR) to spread them over the banks:
//   k contiguous  row r, 8 chunks of 8 k:      chunk c at c ^ ((r & 7) ^ ((r >> 3) & 1))
//   k-major       row k, pieces of 16 columns: piece q at q ^ (2 (k & 3) ^ ((k >> 1) & 1))
#pragma once

#include "rr_common.h"
#include "rr_mfma.h"

namespace rr {
namespace gemm {

constexpr int BK = 64;

struct OpBf16 {};
struct OpF16 {};

template <typename Op>
__device__ __forceinline__ f32x16_t mma(const u16x8_t& a, const u16x8_t& b, f32x16_t c) {
  if constexpr (__is_same(Op, OpBf16)) {
    return mfma32(a, b, c);
  } else {
    typedef _Float16 f16x8_t __attribute__((__vector_size__(16)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  }
}

// fp32 -> the bits of the operand type (round to nearest even).
template <typename Op>
__device__ __forceinline__ uint16_t op_bits(float v) {
  if constexpr (__is_same(Op, OpBf16)) return bf_bits(v);
  else return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}
template <typename Op>
__device__ __forceinline__ float op_val(uint16_t b) {
  if constexpr (__is_same(Op, OpBf16)) return bf_val(b);
  else return static_cast<float>(__builtin_bit_cast(_Float16, b));
}

// One operand of a tile: element (outer o, inner i) at p[o * ld + i]; outside
// o < outer, i < inner it reads as 0.  k contiguous: o = the tile's row, i = k;
// k-major: o = k, i = the tile's column.  ld and inner are multiples of 8, p
// 16-byte aligned.  `plane`: elements from the high to the low plane of an
// operand that is split in two.
struct Operand {
  const uint16_t* p;
  int64_t ld;
  int64_t plane;
  int outer, inner;
};

template <int ROWS, bool KMAJOR>
struct Tile {
  static constexpr int ELEMS = ROWS * BK;
  static constexpr int CHUNKS = ELEMS / 8;
  static constexpr int PER_ROW = KMAJOR ? ROWS / 8 : BK / 8;
  static constexpr int PIECES = ROWS / 16;   // of a k-major row
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (KMAJOR) return ((2 * (row & 3)) ^ ((row >> 1) & 1)) & (PIECES - 1);
    else return (row & 7) ^ ((row >> 3) & 1);
  }
  // Row and chunk column of the chunk that lies at 16-byte position P.
  static __device__ __forceinline__ void at(int P, int& row, int& col) {
    row = P / PER_ROW;
    const int c = P % PER_ROW;
    if constexpr (KMAJOR) col = ((c >> 1) ^ swz(row)) * 2 + (c & 1);
    else col = c ^ swz(row);
  }
  // Fragment of rows (k contiguous) or columns (k-major) r0 .. r0 + 31, k = 16 ks ..:
  // lane l holds row l % 32, k = 8 (l / 32) + e.
  static __device__ __forceinline__ u16x8_t frag32(const uint16_t* t, int r0, int ks, int lane) {
    if constexpr (KMAJOR) {
      const int g = lane >> 4, i = lane & 15;
      const int k = 16 * ks + 8 * (g >> 1) + (i >> 2);
      const int q = (r0 >> 4) + (g & 1);
      const uint16_t* a = t + k * ROWS + (q ^ swz(k)) * 16 + 4 * (i & 3);   // swz(k + 4) = swz(k)
      const u16x4_t lo = tr_read4(a), hi = tr_read4(a + 4 * ROWS);
      return u16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    } else {
      const int r = r0 + (lane & 31);
      const int c = 2 * ks + (lane >> 5);
      return frag(t + r * BK + (c ^ swz(r)) * 8);
    }
  }
};

// WM x WN waves, each with MI x NI blocks of 32 x 32.
template <typename OpT, int BM_, int BN_, int WM_, int WN_, bool AK_, bool BK_MAJOR_>
struct Product {
  using Op = OpT;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int THREADS = 64 * WM * WN;
  static constexpr int MI = BM / WM / 32, NI = BN / WN / 32;
  using TA = Tile<BM, AK_>;
  using TB = Tile<BN, BK_MAJOR_>;
  static constexpr int LDS_ELEMS = TA::ELEMS + TB::ELEMS;
  typedef f32x16_t Acc[MI][NI];

  template <typename T>
  static __device__ __forceinline__ void stage(const Operand& o, const uint16_t* base, int k0, uint16_t* lds, bool kmajor) {
    constexpr int N = T::CHUNKS / THREADS;
    static_assert(T::CHUNKS % THREADS == 0, "every thread stages the same number of chunks");
    u16x8_t v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      int row, col;
      T::at(j * THREADS + (int)threadIdx.x, row, col);
      const int ou = kmajor ? k0 + row : row, in = kmajor ? col * 8 : k0 + col * 8;
      v[j] = u16x8_t{0, 0, 0, 0, 0, 0, 0, 0};
      if (ou < o.outer && in < o.inner) v[j] = *reinterpret_cast<const u16x8_t*>(base + (int64_t)ou * o.ld + in);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) *reinterpret_cast<u16x8_t*>(lds + (j * THREADS + (int)threadIdx.x) * 8) = v[j];
  }

  // k from k0 to k1 (multiples of BK).  PA, PB: the operands' planes; of two times
  // two, the three products that are not below the last bit.
  template <int PA, int PB>
  static __device__ __forceinline__ void run(Acc& acc, const Operand& a, const Operand& b, int k0, int k1,
                                             uint16_t* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / WN, wn = wave % WN;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    uint16_t* la = lds;
    uint16_t* lb = lds + TA::ELEMS;
    for (int seg = 0; seg < PA + PB - 1; ++seg) {   // hi hi, then hi lo, then lo hi
      const uint16_t* pa = a.p + (seg >= PB ? a.plane : 0);
      const uint16_t* pb = b.p + (PB == 2 && seg == 1 ? b.plane : 0);
      for (int k = k0; k < k1; k += BK) {
        __syncthreads();
        stage<TA>(a, pa, k, la, AK_);
        stage<TB>(b, pb, k, lb, BK_MAJOR_);
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks) {
          u16x8_t fa[MI], fb[NI];
#pragma unroll
          for (int i = 0; i < MI; ++i) fa[i] = TA::frag32(la, wm * (BM / WM) + 32 * i, ks, lane);
#pragma unroll
          for (int j = 0; j < NI; ++j) fb[j] = TB::frag32(lb, wn * (BN / WN) + 32 * j, ks, lane);
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mma<Op>(fa[i], fb[j], acc[i][j]);
        }
      }
    }
    __syncthreads();   // the tile's LDS is free
  }
};

}  // namespace gemm
}  // namespace rr
