// rr_gemm.h — the tiled matrix product of the output-head losses on gfx950.
//
// acc[m][n] = sum_k A(m, k) B(n, k) for a BM x BN tile, fp32 accumulation: 16-bit operands
// on the 16x16x32 MFMA, fp32 operands on the fp32 16x16x4 MFMA.  An operand lies in
// memory either with k contiguous (its rows are m or n) or k-major (its rows are k);
// in LDS the tile keeps the orientation it has in memory, and k-major tiles are read
// with the transposing LDS read (fp32: element by element), so no operand is ever
// transposed in memory.
//
// LDS holds 16-byte chunks, a step of 128 bytes of k (64 of 16 bits, 32 of fp32).  A
// fragment read takes the same chunk column of many rows, whose addresses differ by a
// multiple of the row length, so chunk columns are permuted by row (an XOR) to spread
// them over the banks:
//   k contiguous     row r, 8 chunks:              chunk c at c ^ ((r >> 1) & 7)
//   k-major 16 bits  row k, pieces of 16 columns:  piece q at q ^ ((k & 3) + 4 ((k >> 3) & 1))
//   k-major fp32     row k, pieces of 16 columns:  piece q at q ^ ((k >> 2) & 3)
//
// A step is loaded by buffer loads that write LDS themselves (16 bytes a lane,
// the permutation made by the lanes' addresses), into one of two LDS buffers, while the
// other is multiplied.  One barrier a step, behind the first two rows of blocks of its
// second half, says both that the buffer has been read and that the other is full; the
// loads of the step after next follow it, a whole step before they are waited for.
// A fragment of A is read again, for the next half, one row of blocks behind its last
// use, so that reads, loads and products alternate without a pause.
//
// What bounds it: the power limit.  At 8192 x 65536 x 2560 the matrix units are busy
// 65 % of the cycles, at 1.8 of 2.4 GHz; variants with fewer idle cycles ran at a lower
// clock in the same time.  What counts is energy: 16x16x32 products in place of
// 32x32x16 (whose accumulators move twice the bytes a flop) took 2.10 ms in place of
// 2.39, with 4 waves of 128 x 128 in place of 8 of 128 x 64 nothing was won.  LDS reads
// without bank conflicts (half of the LDS cycles before) took 1 % off.
#pragma once

#include "rr_common.h"
#include "rr_mfma.h"

namespace rr {
namespace gemm {

struct OpBf16 {};
struct OpF16 {};
struct OpF32 {};
template <typename Op> constexpr int kBytes = __is_same(Op, OpF32) ? 4 : 2;    // of an element
template <typename Op> constexpr int kStep = 128 / kBytes<Op>;                 // k of a step

template <typename Op>
__device__ __forceinline__ f32x4_t mma(const u16x8_t& a, const u16x8_t& b, f32x4_t c) {
  if constexpr (__is_same(Op, OpBf16)) {
    return mfma16(a, b, c);
  } else if constexpr (__is_same(Op, OpF16)) {
    typedef _Float16 f16x8_t __attribute__((__vector_size__(16)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  } else {   // the e-th product takes k = 4 (lane / 16) + e from both sides
    const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
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

// One operand of a tile: element (outer o, inner i) at byte o * ld + i of p; outside
// o < outer, i < inner it reads as 0.  k contiguous: o = the tile's row, i = k's byte;
// k-major: o = k, i = the column's byte.  ld and inner are multiples of 16, p 16-byte
// aligned.  `plane`: bytes from the high to the low plane of a B that is split in two.
// ld <= 2^22, so that a tile spans at most 2^30 bytes.
struct Operand {
  const void* p;
  int64_t ld;
  int64_t plane;
  int outer, inner;
};

typedef int i32x4_t __attribute__((ext_vector_type(4)));
// 16 bytes a lane from buffer `rsrc` at byte `voff` (0 where that is past its end) to
// LDS byte `lds` + 16 lane.  Not known to the compiler: the reader waits for vmcnt.
__device__ __forceinline__ void load_to_lds(i32x4_t rsrc, int voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds), "v"(voff), "s"(rsrc) : "memory");
}
// What is written before stays before (the compiler would sink the reads to their uses).
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }
// A barrier behind this wave's LDS reads and its loads to LDS.
__device__ __forceinline__ void loads_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_byte(const char* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p);
}

// ROWS rows (k contiguous) or columns (k-major) of a step of elements of EB bytes.
template <int ROWS, bool KMAJOR, int EB>
struct Tile {
  static constexpr int BYTES = ROWS * 128;
  static constexpr int CHUNKS = BYTES / 16;
  static constexpr int PER_ROW = KMAJOR ? ROWS * EB / 16 : 8;
  static constexpr int PIECE = EB;          // chunks of 16 columns of a k-major row
  static constexpr int PIECES = ROWS / 16;
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (!KMAJOR) return (row >> 1) & 7;
    else if constexpr (EB == 2) return ((row & 3) | ((row >> 1) & 4)) & (PIECES - 1);
    else return ((row >> 2) & 3) & (PIECES - 1);
  }
  // Row and chunk column of the chunk that lies at 16-byte position P.
  static __device__ __forceinline__ void at(int P, int& row, int& col) {
    row = P / PER_ROW;
    const int c = P % PER_ROW;
    if constexpr (KMAJOR) col = ((c / PIECE) ^ swz(row)) * PIECE + c % PIECE;
    else col = c ^ swz(row);
  }
  // Fragment of rows (k contiguous) or columns (k-major) r0 .. r0 + 15, half ks of the step:
  // lane l holds row l % 16 and the 16 bytes of k from chunk 4 ks + l / 16.
  static __device__ __forceinline__ u16x8_t frag16(const char* t, int r0, int ks, int lane) {
    const int g = lane >> 4, i = lane & 15;
    if constexpr (!KMAJOR) {
      const int r = r0 + i, c = 4 * ks + g;
      return *reinterpret_cast<const u16x8_t*>(t + r * 128 + (c ^ swz(r)) * 16);
    } else if constexpr (EB == 2) {
      const int k = 32 * ks + 8 * g + (i >> 2);
      const uint16_t* a = reinterpret_cast<const uint16_t*>(t) + k * ROWS + ((r0 >> 4) ^ swz(k)) * 16 + 4 * (i & 3);
      const u16x4_t lo = tr_read4(a), hi = tr_read4(a + 4 * ROWS);   // swz(k + 4) = swz(k)
      return u16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    } else {
      const int k = 16 * ks + 4 * g;
      const float* a = reinterpret_cast<const float*>(t) + k * ROWS + ((r0 >> 4) ^ swz(k)) * 16 + i;
      return __builtin_bit_cast(u16x8_t, f32x4_t{a[0], a[ROWS], a[2 * ROWS], a[3 * ROWS]});   // swz(k + 3) = swz(k)
    }
  }
};

// Bytes of a buffer that starts `skip` bytes into the first of `rows` rows and ends `inner`
// bytes into the last: never negative, which the hardware would take for 4 GiB (a last step
// may start behind the end of an only row).
constexpr __host__ __device__ int buffer_bytes(int rows, int ld, int inner, int skip) {
  const int b = rows <= 0 ? 0 : (rows - 1) * ld + inner - skip;
  return b > 0 ? b : 0;
}
static_assert(buffer_bytes(1, 800, 800, 896) == 0 && buffer_bytes(2, 32, 32, 128) == 0 && buffer_bytes(0, 64, 64, 0) == 0 &&
              buffer_bytes(3, 64, 64, 128) == 64, "a buffer ends with its operand");

// The loads of one operand's tile by the WAVES waves of a workgroup.
template <int ROWS, bool KMAJOR, int EB, int WAVES>
struct Loader {
  using T = Tile<ROWS, KMAJOR, EB>;
  static constexpr int STEP = 128 / EB;                // k of a step
  static constexpr int N = T::CHUNKS / (64 * WAVES);   // loads a thread and step
  static_assert(T::CHUNKS % (64 * WAVES) == 0 && WAVES % 2 == 0, "every thread loads the same number of chunks");
  static constexpr int kPast = 0x40000000;   // beyond any buffer here
  int voff[N];
  int col;          // k contiguous: byte of this thread's chunks in a step
  int ldb, outer, inner;
  const char* at;   // the next step

  __device__ __forceinline__ void init(const Operand& o, int wave, int lane) {
    ldb = (int)o.ld, outer = o.outer, inner = o.inner;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      int row, c;
      T::at((j * WAVES + wave) * 64 + lane, row, c);
      voff[j] = KMAJOR && c * 16 >= inner ? kPast : row * ldb + c * 16;
      col = c * 16;   // k contiguous: the same for every j, WAVES being even
    }
  }
  __device__ __forceinline__ void seek(const void* p, int k) {
    at = static_cast<const char*>(p) + (KMAJOR ? (int64_t)k * ldb : (int64_t)k * EB);
  }
  // The buffer of the step that starts at k, `plane` bytes on, and this thread's offset
  // past its end.
  __device__ __forceinline__ void step(int k, int64_t plane, i32x4_t& r, int& past) const {
    const int rows = KMAJOR ? min(outer - k, STEP) : min(outer, ROWS);
    const int bytes = buffer_bytes(rows, ldb, inner, KMAJOR ? 0 : k * EB);
    const uint64_t b = reinterpret_cast<uint64_t>(at + plane);
    r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32) & 0xffff);
    r[2] = __builtin_amdgcn_readfirstlane(bytes);
    r[3] = 0x00020000;   // raw 32-bit buffer
    past = !KMAJOR && k * EB + col >= inner ? kPast : 0;   // the rest of a last step's row
  }
  __device__ __forceinline__ void advance() { at += KMAJOR ? (int64_t)STEP * ldb : 128; }
  __device__ __forceinline__ void load(int j, i32x4_t r, int past, uint32_t lds, int wave) const {
    load_to_lds(r, voff[j] | past, lds + (uint32_t)(j * WAVES + wave) * 1024);
  }
};

// Tile of workgroup `b` of nm x nn.  Workgroups go to the 8 XCDs in turn, each with an
// L2 of its own: an XCD takes a contiguous part of the tiles, in bands of kBand tiles
// along m walked along n, so that the tiles it multiplies at one time share rows of
// both operands.
constexpr int kXcds = 8, kBand = 8;
__device__ __forceinline__ void tile_of(int b, int nm, int nn, int& m, int& n) {
  const int all = nm * nn, each = all / kXcds, more = all % kXcds;
  const int x = b % kXcds;
  const int id = x * each + min(x, more) + b / kXcds;
  const int band = id / (kBand * nn), in = id - band * kBand * nn;
  const int wide = min(kBand, nm - band * kBand);
  m = band * kBand + in % wide;
  n = in / wide;
}

// WM x WN waves, each with MI x NI blocks of 16 x 16: element e of a lane's block (i, j)
// is row 16 i + 4 (lane / 16) + e and column 16 j + lane % 16 of the wave's part.
template <typename OpT, int BM_, int BN_, int WM_, int WN_, bool AK_, bool BK_MAJOR_>
struct Product {
  using Op = OpT;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int MW = BM / WM, NW = BN / WN;   // a wave's part
  static constexpr int MI = MW / 16, NI = NW / 16;
  static constexpr int EB = kBytes<Op>, BK = kStep<Op>;
  using TA = Tile<BM, AK_, EB>;
  using TB = Tile<BN, BK_MAJOR_, EB>;
  static constexpr int STEP = TA::BYTES + TB::BYTES;
  static constexpr int LDS_BYTES = 2 * STEP;
  static_assert(MI >= 2, "the barrier of a step lies behind the second row of blocks");
  typedef f32x4_t Acc[MI][NI];

  // The step whose loads are under way.
  struct Steps {
    Loader<BM, AK_, EB, WAVES> a;
    Loader<BN, BK_MAJOR_, EB, WAVES> b;
    i32x4_t ra, rb;
    int pa, pb;
    uint32_t lds;
    static constexpr int N = decltype(a)::N + decltype(b)::N;
    __device__ __forceinline__ void load(int j, int wave) const {
      if (j < decltype(a)::N) a.load(j, ra, pa, lds, wave);
      else b.load(j - decltype(a)::N, rb, pb, lds + TA::BYTES, wave);
    }
  };

  // k from k0 to k1 (multiples of BK).  PB: planes of B, each multiplied by A.
  // meanwhile(): what is done while the first loads are under way.
  template <int PB, typename F>
  static __device__ __forceinline__ void run(Acc& acc, const Operand& a, const Operand& b, int k0, int k1, char* lds,
                                             F meanwhile) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int steps = (k1 - k0) / BK * PB;   // the planes' products are made step by step
    if (steps <= 0) {
      meanwhile();
      return;
    }
    Steps st;
    st.a.init(a, wave, lane);
    st.b.init(b, wave, lane);
    st.a.seek(a.p, k0);
    st.b.seek(b.p, k0);
    const uint32_t base = lds_byte(lds);
    int seg = 0, k = k0, loaded = 0;    // the step that is loaded next
    auto next_step = [&] {
      st.lds = base + (uint32_t)(loaded & 1) * STEP;
      st.a.step(k, 0, st.ra, st.pa);
      st.b.step(k, seg == 1 ? b.plane : 0, st.rb, st.pb);
      if (loaded >= steps) st.ra[2] = st.rb[2] = 0;   // behind the last step: loads of nothing (zeros)
      ++loaded;
      if (PB > 1 && ++seg < PB) return;
      seg = 0, k += BK;
      st.a.advance();
      st.b.advance();
    };
    u16x8_t fa[MI], fb[2][NI];
    auto read_a = [&](int i, const char* buf, int ks) { fa[i] = TA::frag16(buf, wm * MW + 16 * i, ks, lane); };
    auto read_b = [&](int j, const char* buf, int ks) { fb[ks][j] = TB::frag16(buf + TA::BYTES, wn * NW + 16 * j, ks, lane); };
    // Row i of the products of k group ks; behind each product act(j).
    auto row = [&](int i, int ks, auto act) {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        acc[i][j] = mma<Op>(fa[i], fb[ks][j], acc[i][j]);
        keep_order();
        act(j);
        keep_order();
      }
    };
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      next_step();
#pragma unroll
      for (int j = 0; j < Steps::N; ++j) st.load(j, wave);
    }
    meanwhile();
    loads_barrier();
#pragma unroll
    for (int i = 0; i < MI; ++i) read_a(i, lds, 0);
#pragma unroll
    for (int j = 0; j < NI; ++j) read_b(j, lds, 0);
    keep_order();
    // A row's fragment of A is read again, for the next k group, one row behind its last
    // use; the fragments of B have a set for each group.
    for (int s = 0; s < steps; ++s) {
      const char* buf = lds + (s & 1) * STEP;
      const char* other = lds + ((s + 1) & 1) * STEP;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        row(i, 0, [&](int j) {
          if (j == 0) {
            if (i == 0) read_a(MI - 1, buf, 0);
            else read_a(i - 1, buf, 1);
          }
          if (j == 1) {
#pragma unroll
            for (int f = i * NI / MI; f < (i + 1) * NI / MI; ++f) read_b(f, buf, 1);
          }
        });
      }
      next_step();
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        row(i, 1, [&](int j) {
          constexpr int R = MI - 1;
          if (i == 0) {
            if (j == 0) read_a(MI - 1, buf, 1);
            return;
          }
          if (j == 0) {
            if (i == 1) loads_barrier();   // the buffer is read, the other full
            read_a(i - 1, other, 0);
          }
          if (j == 1) {
#pragma unroll
            for (int f = (i - 1) * NI / R; f < i * NI / R; ++f) read_b(f, other, 0);
          }
          constexpr int Q = NI < 4 ? 1 : 3;   // products that the loads lie behind
          if (j >= NI - Q) {
            const int q = j - (NI - Q), l0 = (i - 1) * Steps::N / R, l1 = i * Steps::N / R;
#pragma unroll
            for (int l = 0; l < Steps::N; ++l)
              if (l >= l0 + q * (l1 - l0) / Q && l < l0 + (q + 1) * (l1 - l0) / Q) st.load(l, wave);
          }
        });
      }
    }
    loads_barrier();   // the LDS is free
  }

  template <int PB>
  static __device__ __forceinline__ void run(Acc& acc, const Operand& a, const Operand& b, int k0, int k1, char* lds) {
    run<PB>(acc, a, b, k0, k1, lds, [] {});
  }
};

}  // namespace gemm
}  // namespace rr
