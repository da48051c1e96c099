// linear_loss.hip — losses over a large vocabulary straight from hidden states, on
// gfx950: cross entropy on labels and distillation from a teacher's top logits.
//
//   z = h w^T  [rows, V];  s = z / tau;  lse = log sum_v exp(s_v);  q = exp(s - lse)
//   cross entropy (tau = 1)  loss = lse - z_label + zl lse^2
//                            dz = c ((1 + 2 zl lse) q - 1[v = label])
//   distillation             p = softmax over the row's teacher entries of t / tau
//                            loss = tau^2 sum_k p_k (log p_k - log q_{id_k})
//                            dz = c tau (q - sum_{k: id_k = v} p_k)
//   dh = dz w,  dw = dz^T h,  c the row's upstream gradient
//
// A label is a teacher with one entry of weight 1, so both run on the same
// kernels.  The forward forms the logits a tile at a time and keeps each row's running
// maximum and sum per tile and the logits of the row's entries; where that pays
// (kKeepBytes and kKeepChannels below) and the caller has room it also leaves the logits
// themselves, in fp32.
// The backward reads them, or forms them again, a piece of the vocabulary at a time,
// rounds that piece of dz to the operands' 16 bits (for few rows to two planes of them;
// fp32 inputs: not at all), and uses it for dw (complete for the piece) and dh (added
// up over the pieces in fp32).
//
// What bounds it: with many rows the products, two to four of 2 rows V D flops (8192 x
// 65536 x 2560 bf16 forward and backward 7.45 ms, 1.1 PFLOP/s of the three it cannot do
// without; a large product alone runs at 1.4); with few rows the weight's bytes, read
// once forward and once backward and dw's written (16 x 65536 x 5120 bf16 forward 131 us, 5.1
// TB/s, with the backward 545 us, 3.7 TB/s); below about 200 us the launches, 10 to 15.
// Where a product has fewer tiles than CUs its sum is cut in parts that are joined by a
// launch more (best_parts): the logits' over the channels, dh's over the words, dw's over the
// rows (fp32, 209 rows of 3456 channels, 832 words, forward and backward: 543 us whole, 151 cut).
//
// Rows that count for nothing (an ignored label, no teacher entry) are left out
// before the products: the rows that remain are gathered, in order, and their
// number stays on the device.  What such a row's hidden state holds is not read.
//
// fp32 inputs run on the fp32 MFMA, at a ninth of the 16-bit rate, as they are: what a row, a
// word or an upstream gradient gives does not depend on the sizes of the others (1536 x 768 x 32000
// forward and backward 1.83 ms, 124 TFLOP/s of the 153 that a large product reaches).  (Two fp16
// planes an operand, 22 bits below a power of two for the whole tensor, took half the time, but
// hold nothing below 2^-40 of the largest value: one row 1e10 times the others' size put their
// losses off by 0.1, and rare words' rows of dw had a few bits.)
// fp16 dz carries a power of two that brings the largest |dz| just below 2^14, so that
// small probabilities keep their bits; bf16 and fp32 need none.  Where each row has an
// upstream gradient of its own the power is the row's own too: dh's rows are divided by it
// at the end, and dw reads the hidden states divided by it (a copy, for dw sums over rows).
//
// Everything is added up in a fixed order, without atomics.
#include "rr_common.h"
#include "rr_gemm.h"
#include "rr_mfma.h"

#include <algorithm>
#include <string>
#include <type_traits>

namespace {

using rr::bf16;
using rr::f16;
using rr::f32x4_t;
using namespace rr::gemm;

constexpr int kAbsent = 0x7fffffff;
constexpr int64_t kMaxEntries = 1024;      // teacher entries of a row
constexpr int64_t kMaxVocab = 1 << 24;
constexpr int64_t kMaxChannels = 1 << 16;
constexpr int64_t kPieceBytes = (int64_t)512 << 20;   // of dz, where the rows leave room for a piece of kMinPiece
constexpr int64_t kMinPiece = 2048;
constexpr int64_t kPartBytes = (int64_t)256 << 20;    // of the parts that a sum is made in, at most
constexpr int64_t kMaxPiece = 1 << 20;       // a row of a tile's operand is at most so long
constexpr int64_t kFewRows = 64;           // rows whose dz keeps a second plane
constexpr int64_t kKeepRows = 256;         // rows whose logits are always kept
// Logits are kept where they take no more than 4 GiB (of 288) and, with many rows, writing and
// reading one costs less than its product: forward and backward of 1024 x 32000 in bf16 with 768,
// 1024 and 2560 channels 267, 293 and 568 us kept, 266, 298 and 633 formed again; 8192 x 65536
// x 2560 7.6 and 8.9 ms.  fp32 products cost more, so theirs are kept from a twelfth of the
// channels on: 1536 x 32000 with 64, 96 and 192 channels 588, 634 and 680 us kept, 583, 671 and
// 762 formed again.  Few rows' are always kept: their product is a whole reading of the weight.
constexpr int64_t kKeepBytes = (int64_t)4 << 30;
constexpr int64_t kKeepChannels = 896;
constexpr int64_t kKeepChannels1 = 448;    // where the tiles are one round: 512 x 32000 x 768 159 us kept, 163 not,
                                           // 1024 x 4096 x 512 103 and 110, 2048 x 8192 x 256 123 and 115
constexpr int kPad = 64;                   // channels are padded to so many
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Tiles: BM (words, or channels) x BN (rows, or words), WM x WN waves.  Tile256 moves the
// fewest bytes a flop; tiles of 128 x 128 and 256 x 128 were no faster anywhere, not even
// where 256 x 256 leaves CUs without work (1536 x 32000 x 768 forward and backward:
// 294 us, 301 to 307 with them).  Tile64 and Tile32 are for a few rows, whose products are
// bound by the weight's bytes (two workgroups a CU): 16 x 65536 x 5120 forward 137 us, 156
// with Tile256.  fp32 has no tile above Tile64 but for dw: its products are slow enough to hide
// the loads, and small tiles fill the last round (300 x 5003 x 1000 forward and backward 212
// us, 274 with Tile256; 2048 x 32000 x 2048 5.86 and 5.77 ms).
struct Tile256 { static constexpr int BM = 256, BN = 256, WM = 2, WN = 4, THREADS = 512; };
struct Tile64 { static constexpr int BM = 256, BN = 64, WM = 4, WN = 1, THREADS = 256; };
struct Tile32 { static constexpr int BM = 256, BN = 32, WM = 4, WN = 1, THREADS = 256; };
enum Tiles { kTile256, kTile64, kTile32 };
constexpr int kEdge = 256;       // BM of all; buffers hold whole tiles

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// Parts of a caller's buffer, at multiples of 256 bytes (of none, where only its size is asked for).
struct Carve {
  char* base;
  size_t off = 0;
  char* operator()(size_t bytes) {
    char* at = base == nullptr ? nullptr : base + off;
    off += (bytes + 255) / 256 * 256;
    return at;
  }
};

// ------------------------------------------------------------------ state
// What the forward leaves for the backward, in one buffer of the caller's.
struct Header {
  int n;                 // rows that count
};
struct State {
  Header* hdr;
  int* rows;     // [rows] the i-th row that counts
  int* pos;      // [rows] its place there, -1 for a row that does not count
  float* lse2;   // [rows] log2 of the row's sum of exponentials (in the order of `rows`)
  float* loss;   // [rows]
  int* ids;      // [rows][K] the entries' columns, ascending; kAbsent past the last
  float* p;      // [rows][K] their weights
  float* z2;     // [rows][K] their logits, times log2(e) / tau
  float* amax;   // [rows] largest finite |hidden| of a row that counts (fp16)
  char* h;       // [rows][Dp] the hidden states that count, as an operand
  char* w;       // [V][Dp] where the weight is copied
  float* z;      // [rows][Vt] their logits, times log2(e) / tau, where they are kept
};

// ------------------------------------------------------------------ plan
struct Plan {
  int64_t T, D, V;
  int dtype;
  bool fp32;
  int eb;              // bytes of an operand's element
  int planes_z;        // of dz
  bool copy_w;         // the weight is copied: its rows are not whole 16-byte chunks
  int64_t Tp, Dp;      // rows to whole tiles, channels to whole k steps
  int64_t Vt, Dt;      // words and channels to whole tiles
  Tiles rows;          // tiles of the logits and dh (dw: Tile256; with Tile64 5 % slower at 16 to 256 rows)
  int64_t cuts;        // parts of the channels that the logits are added up in
  bool keep_few;       // the forward leaves the logits for the backward whatever the caller's room
  bool keep;           // or where there is room
  // backward
  int64_t Vp;          // columns of a piece (whole tiles)
  int64_t splits;      // parts of a piece's columns that dh is added up in
  int64_t cuts_w;      // parts of the rows that dw is added up in
};
constexpr int64_t kCus = 256;
// Seconds of a k step of a round of tiles, against which the parts' bytes (at 4 TB/s, written and read)
// and a launch are weighed: fp32's at 1.4 us too took 210 us at 300 x 5003 x 1000 forward and backward, 185
// now, 5.4 and 4.9 ms at 4678 x 30720 x 535 (but 694 and 719 us at 512 x 32000 x 768).
constexpr double kStep = 1.4e-6;        // Tile256 of 16 bits (smaller tiles: the weight's bytes)
constexpr double kStepF32 = 3.5e-6;     // Tile64, two a CU
constexpr double kStepF32Dw = 7e-6;     // Tile256
constexpr double kLaunch = 5.6e-6;
// How many parts the k steps of `tiles` tiles are cut in, `slots` workgroups running at one
// time: more parts fill the GPU's rounds better, each at a cost of `part` (in steps), more
// than one at a cost of `more`.  At least 4 of the `all` smallest ranges of k in each, and two or
// more of `bytes` each only up to kPartBytes, which costs little: fp32 513 x 7793 x 118226,
// parts of 466 MiB, took 24.4 ms, 25.1 without; bf16 917 x 13461 x 65552 (460 MiB) 5.80 and 5.62.
int64_t best_parts(int64_t tiles, int64_t slots, double steps, double part, double more, int64_t all, int64_t bytes) {
  const int64_t most = std::min(std::min<int64_t>(64, std::max<int64_t>(4, all) / 4), std::max<int64_t>(1, kPartBytes / bytes));
  int64_t best_n = 1;
  double best = 0;
  for (int64_t n = 1; n <= most; ++n) {
    const double cost = (double)((tiles * n + slots - 1) / slots) * steps / (double)n + (double)n * part + (n > 1 ? more : 0);
    if (best == 0 || cost < best) best = cost, best_n = n;
  }
  return best_n;
}
Plan plan_of(int64_t T, int64_t D, int64_t V, int dtype) {
  Plan p{};
  p.T = T, p.D = D, p.V = V, p.dtype = dtype;
  p.fp32 = dtype == RR_F32;
  p.eb = p.fp32 ? 4 : 2;
  // The rounding of dz to 16 bits averages out over the rows of dw; few rows get a
  // second plane, which costs nothing there (the weight's bytes bound the products).
  p.planes_z = !p.fp32 && T <= kFewRows ? 2 : 1;
  p.copy_w = D * p.eb % 16 != 0;
  p.rows = T <= Tile32::BN ? kTile32 : T <= Tile64::BN || p.fp32 ? kTile64 : kTile256;
  p.Tp = p.rows == kTile32 ? Tile32::BN : up(T, kEdge), p.Dp = up(D, kPad);
  p.Vt = up(V, kEdge), p.Dt = up(D, kEdge);
  const int64_t slots = p.rows == kTile256 ? kCus : 2 * kCus;   // workgroups at one time
  const int64_t row_tiles = p.rows == kTile256 ? p.Tp / 256 : p.rows == kTile64 ? up(T, 64) / 64 : 1;
  // Few tiles of many channels: their sums are cut in parts, each at the cost of writing
  // and reading the logits in fp32, and all at that of one launch more.
  const double step = p.fp32 ? kStepF32 : kStep;
  {
    const int64_t all = p.Dp * p.eb / 128;
    const double part = (double)(T * V * 8) / 4e12 / step;
    p.cuts = best_parts(p.Vt / kEdge * row_tiles, slots, (double)all, part, kLaunch / step, all, T * p.Vt * 4);
  }
  const int64_t z_bytes = T * p.Vt * 4;
  p.keep_few = T <= kKeepRows || p.cuts > 1;   // (parts are small, and summed once for both)
  p.keep = p.keep_few ||
           (z_bytes <= kKeepBytes &&
            D * (p.fp32 ? 12 : 1) >= (p.Vt / kEdge * row_tiles <= kCus ? kKeepChannels1 : kKeepChannels));
  const int64_t most = std::min(kMaxPiece, std::max(kMinPiece, kPieceBytes / (p.Tp * p.eb * p.planes_z) / kEdge * kEdge));
  const int64_t pieces = (p.Vt + most - 1) / most;
  p.Vp = up((p.Vt + pieces - 1) / pieces, kEdge);
  // dh has few tiles: its sum over the piece's columns is cut in parts, as the logits' is.
  const int64_t all = p.Vp * p.eb / 128;
  p.splits = best_parts(p.Dt / kEdge * row_tiles, slots, (double)(all * p.planes_z),
                        (double)(T * D * 8) / 4e12 / step, 0., all, p.Tp * p.Dt * 4);
  // Few words and many rows: so is dw's sum over the rows (few rows are few steps).
  p.cuts_w = 1;
  if (T > kKeepRows) {
    const int64_t steps = up(T * p.eb, 128) / 128;
    const double step_w = p.fp32 ? kStepF32Dw : kStep;
    p.cuts_w = best_parts(p.Dt / kEdge * (p.Vp / kEdge), kCus, (double)steps, (double)(p.Vp * D * 8) / 4e12 / step_w,
                          kLaunch / step_w, steps, p.Vp * p.Dt * 4);
  }
  return p;
}

// grad: 0 no backward, 1 logits where they are kept, 2 only those that always are.
size_t state_layout(const Plan& p, int64_t K, int grad, char* base, State* s) {
  Carve take{base};
  State t;
  t.hdr = reinterpret_cast<Header*>(take(sizeof(Header)));
  t.rows = reinterpret_cast<int*>(take((size_t)p.T * 4));
  t.pos = reinterpret_cast<int*>(take((size_t)p.T * 4));
  t.lse2 = reinterpret_cast<float*>(take((size_t)p.T * 4));
  t.loss = reinterpret_cast<float*>(take((size_t)p.T * 4));
  t.ids = reinterpret_cast<int*>(take((size_t)p.T * K * 4));
  t.p = reinterpret_cast<float*>(take((size_t)p.T * K * 4));
  t.z2 = reinterpret_cast<float*>(take((size_t)p.T * K * 4));
  t.amax = reinterpret_cast<float*>(take(p.dtype == RR_F16 ? (size_t)p.T * 4 : 0));
  t.h = take((size_t)p.T * p.Dp * p.eb);
  t.w = take(p.copy_w ? (size_t)p.V * p.Dp * p.eb : 0);
  const bool keep = grad == 1 ? p.keep : grad == 2 && p.keep_few;
  t.z = reinterpret_cast<float*>(take(keep ? (size_t)p.T * p.Vt * 4 : 0));
  if (!keep) t.z = nullptr;
  if (s != nullptr) *s = t;
  return take.off;
}

struct FwdWs {
  float2* part;    // [word tiles][Tp] maximum and sum of a tile's row
  float* cut;      // [cuts][T][Vt] parts of the logits, where there are two or more
};
size_t fwd_layout(const Plan& p, char* base, FwdWs* s) {
  Carve take{base};
  FwdWs t;
  t.part = reinterpret_cast<float2*>(take((size_t)(p.Vt / kEdge) * p.Tp * sizeof(float2)));
  t.cut = reinterpret_cast<float*>(take(p.cuts > 1 ? (size_t)p.cuts * p.T * p.Vt * 4 : 0));
  if (s != nullptr) *s = t;
  return take.off;
}
struct BwdWs {
  float* scale;    // the factors on dw and on dh
  float2* coef;    // [Tp] a row's factors (coef_kernel)
  float* unscale;  // [Tp] the inverse of a row's power of two (fp16)
  char* h;         // [T][Dp] the hidden states times that (fp16)
  char* dz;        // [planes_z][Tp][Vp]
  float* dh;       // [splits][Tp][Dt]
  float* dw;       // [cuts_w][Vp][Dt], where there are two or more
};
size_t bwd_layout(const Plan& p, char* base, BwdWs* s) {
  Carve take{base};
  BwdWs t;
  t.scale = reinterpret_cast<float*>(take(256));
  t.coef = reinterpret_cast<float2*>(take((size_t)p.Tp * sizeof(float2)));
  t.unscale = reinterpret_cast<float*>(take(p.dtype == RR_F16 ? (size_t)p.Tp * 4 : 0));
  t.h = take(p.dtype == RR_F16 ? (size_t)p.T * p.Dp * p.eb : 0);
  t.dz = take((size_t)p.planes_z * p.Tp * p.Vp * p.eb);
  t.dh = reinterpret_cast<float*>(take((size_t)p.splits * p.Tp * p.Dt * 4));
  t.dw = reinterpret_cast<float*>(take(p.cuts_w > 1 ? (size_t)p.cuts_w * p.Vp * p.Dt * 4 : 0));
  if (s != nullptr) *s = t;
  return take.off;
}

// ------------------------------------------------------------------ rows and entries
// A power of two that brings a largest value of these bits into [2^(e - 1), 2^e)
// (1 where there is none), both it and its inverse a normal value.
__device__ __forceinline__ float pow2_to(uint32_t amax_bits, int e) {
  if (amax_bits == 0) return 1.f;
  const int x = (int)(amax_bits >> 23) - 127;   // floor(log2) of a normal value
  return ldexpf(1.f, max(-126, min(126, e - 1 - x)));
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// A row's teacher entries by column (a wave per row): ids ascending, absent ones
// (id < 0 or a logit of -inf) last, and their softmax weights: the temperature divides
// differences of logits, which a large one of the type's range outlasts.  The id of an entry past
// the vocabulary makes the row's weights, and with them its loss and gradients, NaN.
// pos[row] = 1 where the row has an entry.
template <typename E>
__global__ void __launch_bounds__(64)
entries_kernel(const E* __restrict__ logits, const int64_t* __restrict__ ids_in, int K, int KP, int V, float tau,
               int* __restrict__ ids, float* __restrict__ p, int* __restrict__ pos) {
  extern __shared__ char sm[];
  int* id = reinterpret_cast<int*>(sm);
  float* t = reinterpret_cast<float*>(sm) + KP;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  float worst = 0.f;   // NaN: an id past the vocabulary
  for (int k = lane; k < KP; k += 64) {
    int i = kAbsent;
    float v = -INFINITY;
    if (k < K) {
      const int64_t raw = ids_in[row * K + k];
      const float x = rr::to_f32(logits[row * K + k]);
      if (raw >= 0 && x != -INFINITY) {
        if (raw < V) i = (int)raw, v = x;
        else worst = NAN;
      }
    }
    id[k] = i, t[k] = v;
  }
  __syncthreads();
  for (int size = 2; size <= KP; size *= 2)
    for (int step = size / 2; step > 0; step /= 2) {
      for (int k = lane; k < KP / 2; k += 64) {
        const int a = 2 * k - (k & (step - 1)), b = a + step;
        const bool asc = (a & size) == 0;
        const int ia = id[a], ib = id[b];
        if ((ia > ib) == asc && ia != ib) {
          const float ta = t[a], tb = t[b];
          id[a] = ib, id[b] = ia, t[a] = tb, t[b] = ta;
        }
      }
      __syncthreads();
    }
  float m = -INFINITY;
  for (int k = lane; k < K; k += 64) m = fmaxf(m, t[k]);
  m = wave_max(m);
  const bool any = id[0] != kAbsent;
  float s = 0.f;
  for (int k = lane; k < K; k += 64)
    if (id[k] != kAbsent) s += expf((t[k] - m) / tau);
  s = wave_add(s) + wave_add(worst);
  for (int k = lane; k < K; k += 64) {
    ids[row * K + k] = id[k];
    p[row * K + k] = id[k] != kAbsent ? expf((t[k] - m) / tau) / s : s != s ? NAN : 0.f;
  }
  if (lane == 0) pos[row] = any || s != s ? 1 : 0;
}

// The rows that count, in order (one workgroup).  Labels: `labels` decides, and
// their entries are written here; an invalid label is an absent entry of weight
// NaN.  Teacher: pos holds what entries_kernel found.
template <bool LABELS>
__global__ void __launch_bounds__(1024)
rows_kernel(const int64_t* __restrict__ labels, int64_t ignore, int64_t T, int V, State st) {
  __shared__ int sums[16];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  int base = 0;
  for (int64_t i0 = 0; i0 < T; i0 += 1024) {
    const int64_t i = i0 + tid;
    bool in = false;
    if (i < T) {
      if constexpr (LABELS) {
        const int64_t l = labels[i];
        in = l != ignore;
        const bool ok = l >= 0 && l < V;
        st.ids[i] = ok ? (int)l : kAbsent;
        st.p[i] = ok || !in ? 1.f : NAN;
      } else {
        in = st.pos[i] != 0;
      }
    }
    const uint64_t b = __ballot(in);
    const int before = __popcll(b & ((1ull << lane) - 1));
    __syncthreads();   // the last turn's reads of sums are done
    if (lane == 0) sums[wave] = __popcll(b);
    __syncthreads();
    int at = base, all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) at += sums[w];
      all += sums[w];
    }
    at += before;
    if (i < T) {
      st.pos[i] = in ? at : -1;
      if (in) st.rows[at] = (int)i;
      if (!in) st.loss[i] = 0.f;
    }
    base += all;
  }
  if (tid == 0) st.hdr->n = base;
}

// Eight elements from column c of a row of D as they lie in memory, 0 past its end (a row
// may start at any element).
template <typename X>
__device__ __forceinline__ void load8(const X* row, int c, int D, X (&v)[8]) {
  if (c + 8 <= D) {
    typedef uint32_t Words __attribute__((ext_vector_type(2 * sizeof(X))));
    typedef Words Any __attribute__((aligned(sizeof(X))));
    const Words w = *reinterpret_cast<const Any*>(row + c);
    __builtin_memcpy(v, &w, sizeof(w));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < D ? row[c + e] : X{};
  }
}

// The hidden states that count (blockIdx.y = 0) and the weight (1) as operands: copied, padded
// with zeros to Dp channels.  fp16: and the largest finite |hidden| of each row.
template <typename X>
__global__ void __launch_bounds__(256)
pack_kernel(const X* __restrict__ hidden, const X* __restrict__ weight, int64_t V, int D, int Dp, State st) {
  const bool w = blockIdx.y == 1;
  const X* x = w ? weight : hidden;
  const int* rows = w ? nullptr : st.rows;
  const int64_t n = w ? V : st.hdr->n;
  X* out = reinterpret_cast<X*>(w ? st.w : st.h);
  __shared__ float buf[4];
  for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
    const X* xr = x + (rows != nullptr ? (int64_t)rows[r] : r) * D;
    float m = 0.f;
    for (int c = threadIdx.x * 8; c < Dp; c += 2048) {
      X v[8];
      load8(xr, c, D, v);
      if constexpr (__is_same(X, f16)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = fabsf(rr::to_f32(v[e]));
          if (a < INFINITY) m = fmaxf(m, a);   // neither infinite nor NaN
        }
      }
      typedef uint32_t Words __attribute__((ext_vector_type(2 * sizeof(X))));
      Words q;
      __builtin_memcpy(&q, v, sizeof(q));
      *reinterpret_cast<Words*>(out + r * Dp + c) = q;
    }
    if constexpr (__is_same(X, f16)) {
      if (w) continue;
      m = wave_max(m);
      __syncthreads();   // the last row's reads of buf are done
      if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = m;
      __syncthreads();
      if (threadIdx.x == 0) st.amax[r] = fmaxf(fmaxf(buf[0], buf[1]), fmaxf(buf[2], buf[3]));
    }
  }
}

// ------------------------------------------------------------------ logits
// (row lengths and planes of operands in bytes)
struct LogitArgs {
  const char* w;          // [V][ldw]
  const char* h;          // [n][Dp]
  int64_t ldw, ldh;
  int V, Dp, K, Tp, nvt;  // nvt: tiles of this launch
  float c;                // log2(e) / tau
  State st;
  float2* part;           // forward
  float* z;               // forward: [n][ldzf] logits that are kept, or [cuts][ldcut] parts of them
  int64_t ldzf, ldcut;
  int cuts;
  const float2* coef;     // backward
  char* dz;
  int64_t ldz, plane_z;
  int v_first;            // the piece's first column
};

// A logit in units of log2 is rounded before the maximum or lse is taken off: fused into
// one operation, a logit would not be 0 off itself, and a sure word's probability not 1.
__device__ __forceinline__ float rounded(float x) {
  asm("" : "+v"(x));
  return x;
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// First of a row's K entries at column v0 or behind.
__device__ __forceinline__ int first_entry(const int* ids, int K, int v0) {
  int lo = 0, hi = K;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ids[mid] < v0) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}
// Walks a row's entries from the lo-th on that lie in this wave's columns v0 .. v0 + 16 MI
// and in this lane's quarter of the accumulator rows: f(k, element) with the element's
// index 4 i + e.
template <int MI, typename F>
__device__ __forceinline__ void each_entry(const int* ids, int K, int lo, int v0, int quarter, F f) {
  for (int k = lo; k < K; ++k) {
    const int rel = ids[k] - v0;
    if (rel >= 16 * MI) break;
    if (((rel >> 2) & 3) == quarter) f(k, (rel >> 4) * 4 + (rel & 3));
  }
}

// One of a wave's column blocks (16 rows of the output, MW consecutive values of each) to
// memory through LDS, so that a row leaves in whole lines: value(i) is the lane's four of
// block i (its row lane % 16, from 16 i + 4 (lane / 16)), store(r, c, v) takes 16 bytes of
// row r from value c on.  `lds`: 16 (MW + 16 / sizeof(T)) values of the wave's own.
template <int MI, typename T, typename F, typename S>
__device__ __forceinline__ void store_block(T* lds, int lane, F value, S store) {
  constexpr int MW = 16 * MI, VEC = 16 / sizeof(T), PITCH = MW + VEC, PER_ROW = MW / VEC;
  typedef T Four __attribute__((ext_vector_type(4)));
  typedef T Vec __attribute__((ext_vector_type(VEC)));
#pragma unroll
  for (int i = 0; i < MI; ++i) *reinterpret_cast<Four*>(lds + (lane & 15) * PITCH + 16 * i + 4 * (lane >> 4)) = value(i);
  rr::wave_lds_sync();
#pragma unroll
  for (int q = 0; q < 16 * PER_ROW / 64; ++q) {
    const int r = q * (64 / PER_ROW) + lane / PER_ROW, c = lane % PER_ROW * VEC;
    store(r, c, *reinterpret_cast<const Vec*>(lds + r * PITCH + c));
  }
  rr::wave_lds_sync();
}

// z^T tiles: m = vocabulary, n = rows, so that a lane holds 4 MI logits of a row.
// kStats: the forward's maxima and sums, and the logits where they are kept; kCut: one part of
// the sums, as it is; kGrad: the backward's dz.
enum Mode { kStats, kCut, kGrad };
template <typename C, typename Op, Mode MODE, int PZ>
__global__ void __launch_bounds__(C::THREADS, 2)
logits_kernel(LogitArgs a) {
  constexpr bool GRAD = MODE == kGrad;
  constexpr int BM = C::BM, BN = C::BN;
  using P = Product<Op, BM, BN, C::WM, C::WN, false, false>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  const int n = a.st.hdr->n;
  int vt, tt;
  int k0 = 0, k1 = a.Dp, cut = 0;
  if constexpr (MODE == kCut) {
    const int tiles = gridDim.x / a.cuts, steps = a.Dp / P::BK;
    cut = blockIdx.x / tiles;
    k0 = steps * cut / a.cuts * P::BK, k1 = steps * (cut + 1) / a.cuts * P::BK;
    tile_of(blockIdx.x - cut * tiles, a.nvt, tiles / a.nvt, vt, tt);
  } else {
    tile_of(blockIdx.x, a.nvt, gridDim.x / a.nvt, vt, tt);
  }
  const int t0 = tt * BN, v0 = a.v_first + vt * BM;
  if (t0 >= n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / P::WN, wn = wave % P::WN;
  const int quarter = lane >> 4;

  typename P::Acc acc;
  const Operand A{a.w + (int64_t)v0 * a.ldw, a.ldw, 0, a.V - v0, (int)a.ldw};
  const Operand B{a.h + (int64_t)t0 * a.ldh, a.ldh, 0, n - t0, (int)a.ldh};
  // What the rows need, looked up while the first loads are under way.
  const int vw = v0 + wm * P::MW, left = a.V - vw;   // the wave's words, and how many there are
  int orig[P::NI];   // first of the row's entries
  int lo[P::NI];     // first of them in the wave's words
  float2 co[P::NI];
  float l2[P::NI];
  P::template run<1>(acc, A, B, k0, k1, lds, [&] {
    if constexpr (MODE == kCut) return;
#pragma unroll
    for (int j = 0; j < P::NI; ++j) {
      const int t = min(t0 + wn * P::NW + 16 * j + (lane & 15), n - 1);
      orig[j] = a.st.rows[t] * a.K;
      if constexpr (GRAD) co[j] = a.coef[t], l2[j] = a.st.lse2[t];
    }
#pragma unroll
    for (int j = 0; j < P::NI; ++j)
      lo[j] = t0 + wn * P::NW + 16 * j + (lane & 15) < n ? first_entry(a.st.ids + orig[j], a.K, vw) : a.K;
  });

  float* fstage = reinterpret_cast<float*>(lds) + wave * 16 * (P::MW + 4);
  float* red = reinterpret_cast<float*>(lds) + P::WAVES * 16 * (P::MW + 4);   // forward: [WM][BN][2]
  static_assert((P::WAVES * 16 * (P::MW + 4) + P::WM * BN * 2) * 4 <= P::LDS_BYTES, "a tile's results go through its LDS");
  auto store_z = [&](int j) {
    const int t = t0 + wn * P::NW + 16 * j;
    float* o = a.z + cut * a.ldcut + (int64_t)t * a.ldzf + vw;
    store_block<P::MI>(fstage, lane, [&](int i) { return acc[i][j]; }, [&](int r, int v, f32x4_t x) {
      if (t + r < n) *reinterpret_cast<f32x4_t*>(o + (int64_t)r * a.ldzf + v) = x;
    });
  };
  if constexpr (MODE == kCut) {
#pragma unroll
    for (int j = 0; j < P::NI; ++j) store_z(j);
    return;
  }
#pragma unroll
  for (int j = 0; j < P::NI; ++j) {
    const int tl = wn * P::NW + 16 * j + (lane & 15);
    const bool on = t0 + tl < n;
    const int* ids = a.st.ids + orig[j];
#pragma unroll
    for (int i = 0; i < P::MI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = rounded(acc[i][j][e] * a.c);
    if (left < P::MW) {   // the vocabulary's last words
#pragma unroll
      for (int i = 0; i < P::MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = 16 * i + 4 * quarter + e < left ? acc[i][j][e] : -INFINITY;
    }
    if constexpr (!GRAD) {
      float m = -INFINITY, part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < P::MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = fmaxf(m, acc[i][j][e]);
#pragma unroll
      for (int i = 0; i < P::MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[e] += exp2_fast(acc[i][j][e] - m);
      float s = (part[0] + part[1]) + (part[2] + part[3]);
      if (m == -INFINITY) {   // no column of the vocabulary, or NaN among the logits
        bool bad = false;
#pragma unroll
        for (int i = 0; i < P::MI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) bad |= acc[i][j][e] != acc[i][j][e];
        s = bad ? NAN : 0.f;
      }
      each_entry<P::MI>(ids, a.K, lo[j], vw, quarter, [&](int k, int el) {
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < P::MI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) z = el == i * 4 + e ? acc[i][j][e] : z;
        a.st.z2[orig[j] + k] = z;
      });
      // the other quarters' words of the same row, then the waves along m
#pragma unroll
      for (int o = 16; o < 64; o *= 2) {
        const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
        const float mm = fmaxf(m, m2);
        s = (m == mm ? s : s * exp2_fast(m - mm)) + (m2 == mm ? s2 : s2 * exp2_fast(m2 - mm));
        m = mm;
      }
      if (quarter == 0) {
        red[(wm * BN + tl) * 2] = m;
        red[(wm * BN + tl) * 2 + 1] = s;
      }
      if (a.z != nullptr) store_z(j);
    } else {
#pragma unroll
      for (int i = 0; i < P::MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = exp2_fast(acc[i][j][e] - l2[j]);   // 0 behind the last word
      // q - p first, so that what is left of a sure label keeps its bits
      each_entry<P::MI>(ids, a.K, lo[j], vw, quarter, [&](int k, int el) {
        const float p = a.st.p[orig[j] + k], r = p * co[j].y;
#pragma unroll
        for (int i = 0; i < P::MI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = el == i * 4 + e ? acc[i][j][e] - p + r : acc[i][j][e];
      });
#pragma unroll
      for (int i = 0; i < P::MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = on ? co[j].x * acc[i][j][e] : 0.f;
      if (left < P::MW) {   // not 0 x NaN
#pragma unroll
        for (int i = 0; i < P::MI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = 16 * i + 4 * quarter + e < left ? acc[i][j][e] : 0.f;
      }
      using Bits = typename std::conditional<P::EB == 4, float, uint16_t>::type;
      typedef Bits Four __attribute__((ext_vector_type(4)));
      typedef Bits Vec __attribute__((ext_vector_type(16 / P::EB)));
      Bits* stage = reinterpret_cast<Bits*>(lds) + wave * 16 * (P::MW + 16 / P::EB);
      char* o = a.dz + (int64_t)(t0 + wn * P::NW + 16 * j) * a.ldz + (vw - a.v_first) * P::EB;
      auto store = [&](int r, int v, Vec x) { *reinterpret_cast<Vec*>(o + (int64_t)r * a.ldz + v * P::EB) = x; };
      store_block<P::MI>(stage, lane, [&](int i) {
        if constexpr (P::EB == 4) return acc[i][j];
        else return Four{op_bits<Op>(acc[i][j][0]), op_bits<Op>(acc[i][j][1]), op_bits<Op>(acc[i][j][2]), op_bits<Op>(acc[i][j][3])};
      }, store);
      if constexpr (PZ == 2) {
        o += a.plane_z;
        store_block<P::MI>(stage, lane, [&](int i) {
          Four lo;
#pragma unroll
          for (int e = 0; e < 4; ++e) lo[e] = op_bits<Op>(acc[i][j][e] - op_val<Op>(op_bits<Op>(acc[i][j][e])));
          return lo;
        }, store);
      }
    }
  }
  if constexpr (!GRAD) {
    __syncthreads();
    for (int tl = threadIdx.x; tl < BN; tl += P::THREADS) {
      float m = -INFINITY, s = 0.f;
      for (int w = 0; w < P::WM; ++w) m = fmaxf(m, red[(w * BN + tl) * 2]);
      for (int w = 0; w < P::WM; ++w) {
        const float mw = red[(w * BN + tl) * 2], sw = red[(w * BN + tl) * 2 + 1];
        s += mw == m ? sw : sw * exp2_fast(mw - m);
      }
      a.part[(int64_t)vt * a.Tp + t0 + tl] = make_float2(m, s);
    }
  }
}

constexpr int kSeg = 2048;   // words of a row that a workgroup of the two kernels below takes, eight a thread

// The parts of the logits added up: what kStats does for a tile, for a segment of a row.
// Bound by the parts' bytes, or its launch.  The segment goes through LDS, so that an entry
// is found by a thread of its own (each thread walking the row's 64 entries: 63 us at 3623 x
// 865 words, 12 now).
__global__ void __launch_bounds__(256)
join_kernel(State st, const float* __restrict__ cut, int cuts, int64_t ldcut, int V, int64_t Vt, int K, float c, int64_t Tp,
             float2* __restrict__ part) {
  __shared__ float red[2][4];
  __shared__ f32x4_t seg[kSeg / 4];
  const int t = blockIdx.x;
  if (t >= st.hdr->n) return;
  const int tid = threadIdx.x, v0 = blockIdx.y * kSeg, v = v0 + tid * 8;
  float z[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] = 0.f;
  if (v < Vt) {   // Vt is a multiple of 8
    const float* at = cut + (int64_t)t * Vt + v;
#pragma unroll 4
    for (int i = 0; i < cuts; ++i) {
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(at + i * ldcut), y = *reinterpret_cast<const f32x4_t*>(at + i * ldcut + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] += x[e], z[4 + e] += y[e];
    }
  }
  float m = -INFINITY, s = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    z[e] = v + e < V ? rounded(z[e] * c) : -INFINITY;
    m = fmaxf(m, z[e]);
  }
  if (st.z != nullptr && v < Vt) {
    float* o = st.z + (int64_t)t * Vt + v;
    *reinterpret_cast<f32x4_t*>(o) = f32x4_t{z[0], z[1], z[2], z[3]};
    *reinterpret_cast<f32x4_t*>(o + 4) = f32x4_t{z[4], z[5], z[6], z[7]};
  }
  seg[2 * tid] = f32x4_t{z[0], z[1], z[2], z[3]}, seg[2 * tid + 1] = f32x4_t{z[4], z[5], z[6], z[7]};
  m = wave_max(m);
  if ((tid & 63) == 0) red[0][tid >> 6] = m;
  __syncthreads();
  const int64_t orig = (int64_t)st.rows[t] * K;
  for (int k = tid; k < K; k += 256) {
    const int rel = st.ids[orig + k] - v0;
    if (rel >= 0 && rel < kSeg) st.z2[orig + k] = reinterpret_cast<const float*>(seg)[rel];
  }
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  if (m != -INFINITY) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s += exp2_fast(z[e] - m);
  } else {   // NaN among the logits
#pragma unroll
    for (int e = 0; e < 8; ++e) s = z[e] != z[e] ? NAN : s;
  }
  s = wave_add(s);
  if ((tid & 63) == 0) red[1][tid >> 6] = s;
  __syncthreads();
  if (tid == 0) part[(int64_t)blockIdx.y * Tp + t] = make_float2(m, (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]));
}

// dz from the logits that were kept: what kGrad does for a tile, for a segment of a row (as
// in join_kernel).  A word's entries are taken off in their order by the thread of the first.
template <typename Op, int PZ>
__global__ void __launch_bounds__(256)
dz_kernel(State st, const float2* __restrict__ coef, int V, int64_t Vt, int K, int v_first, int cols, char* __restrict__ dz,
          int64_t ldz, int64_t plane_z) {
  const int t = blockIdx.x;
  if (t >= st.hdr->n) return;
  const int tid = threadIdx.x, rel0 = blockIdx.y * kSeg, at = rel0 + tid * 8, v0 = v_first + rel0, v = v0 + tid * 8;
  const bool here = at < cols;   // both multiples of 8
  const float2 co = coef[t];
  const float l2 = st.lse2[t];
  __shared__ f32x4_t seg[kSeg / 4];
  if (here) {
    const f32x4_t* i = reinterpret_cast<const f32x4_t*>(st.z + (int64_t)t * Vt + v);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const f32x4_t x = i[q];
      seg[2 * tid + q] = f32x4_t{exp2_fast(x[0] - l2), exp2_fast(x[1] - l2), exp2_fast(x[2] - l2), exp2_fast(x[3] - l2)};
    }
  }
  __syncthreads();
  const int64_t orig = (int64_t)st.rows[t] * K;
  const int* ids = st.ids + orig;
  for (int k = tid; k < K; k += 256) {
    const int id = ids[k], rel = id - v0;
    if (rel < 0 || rel >= min(kSeg, cols - rel0) || (k > 0 && ids[k - 1] == id)) continue;
    float q = reinterpret_cast<float*>(seg)[rel];
    for (int j = k; j < K && ids[j] == id; ++j) {   // a word's entries
      const float p = st.p[orig + j];
      q = q - p + p * co.y;
    }
    reinterpret_cast<float*>(seg)[rel] = q;
  }
  __syncthreads();
  if (!here) return;
  float z[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] = v + e < V ? co.x * reinterpret_cast<const float*>(seg)[8 * tid + e] : 0.f;
  char* o = dz + t * ldz + (int64_t)at * kBytes<Op>;
  if constexpr (kBytes<Op> == 4) {
    reinterpret_cast<f32x4_t*>(o)[0] = f32x4_t{z[0], z[1], z[2], z[3]};
    reinterpret_cast<f32x4_t*>(o)[1] = f32x4_t{z[4], z[5], z[6], z[7]};
  } else {
    rr::u16x8_t hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[e] = op_bits<Op>(z[e]);
      lo[e] = op_bits<Op>(z[e] - op_val<Op>(hi[e]));
    }
    *reinterpret_cast<rr::u16x8_t*>(o) = hi;
    if constexpr (PZ == 2) *reinterpret_cast<rr::u16x8_t*>(o + plane_z) = lo;
  }
}

// Per row (a wave each): the tiles' maxima and sums to the row's lse, and its loss.
__global__ void __launch_bounds__(256)
row_loss_kernel(State st, const float2* __restrict__ part, int nvt, int64_t Tp, int K, bool labels, float zl, float tau,
                float* __restrict__ out) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= st.hdr->n) return;
  const int64_t row = st.rows[t];
  float m = -INFINITY, s = 0.f;
  for (int v = lane; v < nvt; v += 64) {
    const float2 x = part[(int64_t)v * Tp + t];
    const float mm = fmaxf(m, x.x);
    s = (m == mm ? s : s * exp2f(m - mm)) + (x.x == mm ? x.y : x.y * exp2f(x.x - mm));
    m = mm;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
    const float mm = fmaxf(m, m2);
    s = (m == mm ? s : s * exp2f(m - mm)) + (m2 == mm ? s2 : s2 * exp2f(m2 - mm));
    m = mm;
  }
  const float l2 = m + log2f(s);
  float loss = 0.f;
  for (int k = lane; k < K; k += 64) {
    const float p = st.p[row * K + k];
    if (p == 0.f) continue;
    if (st.ids[row * K + k] == kAbsent) {   // an id outside the vocabulary
      loss = NAN;
      continue;
    }
    const float logq = (st.z2[row * K + k] - l2) * kLn2;
    loss += labels ? -logq : p * (logf(p) - logq);
  }
  loss = wave_add(loss);
  if (labels) {
    const float lse = l2 * kLn2;
    loss += zl * lse * lse;
  } else {
    loss *= tau * tau;
  }
  if (lane == 0) {
    out[row] = loss;
    st.lse2[t] = loss != loss ? NAN : l2;   // the backward's row is NaN where the loss is
  }
}

// The sum of the rows' losses, over the number that count where `mean` (0 without any).  A
// launch of its own: the fences by which row_loss_kernel's last workgroup could do it
// took 160 us at 8192 rows.
__global__ void __launch_bounds__(1024)
sum_loss_kernel(const float* __restrict__ loss, int64_t T, const Header* hdr, bool mean, float* out) {
  __shared__ float buf[16];
  float s = 0.f;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < T; i += 1024) s += loss[i];
  s = wave_add(s);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = 0.f;
  for (int w = 0; w < 16; ++w) s += buf[w];
  out[0] = mean ? s / (float)max(1, hdr->n) : s;
}

// ------------------------------------------------------------------ gradients
// coef[t] = (c f, 1 - 1 / f) with f = 1 + 2 zl lse, so that a row of dz is
// c f (q - p + p (1 - 1 / f)), and the factors on dw and dh, scale[0] and [1].  One upstream
// gradient for all rows goes into that factor and c = 1: -1 at a label is exact in 16
// bits, where -c would be off by the same rounding in every row.  Otherwise c is the
// row's.  `scaled`: c carries the power of two that brings the largest of them below
// 2^14, and the factors its inverse; or each row's own does, whose inverse is left in
// unscale (0 where dz is 0), and dw's factor undoes that of the copy of the hidden states
// (scale_h_kernel), which brings the largest of those below 2^15.  One workgroup.
__global__ void __launch_bounds__(1024)
coef_kernel(State st, const float* __restrict__ dloss, bool per_row, bool mean, float factor, float zl, bool scaled,
            float2* __restrict__ coef, float* __restrict__ unscale, float* scale) {
  __shared__ float buf[16];
  const int n = st.hdr->n;
  const bool each = scaled && per_row;
  float m = 0.f;
  for (int t = threadIdx.x; t < n; t += 1024) {
    const float c = per_row ? dloss[st.rows[t]] * factor : 1.f;
    const float x = 2.f * zl * st.lse2[t] * kLn2;
    float f = 1.f + x;
    if (f == 0.f) f = 1e-30f;
    const float a = fmaxf(fabsf(c * f), fabsf(c));   // |dz| <= 2 a
    float sc = 1.f, v = a;
    if (each) {
      float un = 1.f;
      if (a < INFINITY) sc = pow2_to(__float_as_uint(a), 14), un = a == 0.f ? 0.f : 1.f / sc;
      unscale[t] = un;
      v = st.amax[t] * un;
    }
    coef[t] = make_float2(c * f * sc, x / f);
    if (v < INFINITY) m = fmaxf(m, v);
  }
  float sc = 1.f;
  if (scaled) {   // the same for the whole workgroup
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = m;
    __syncthreads();
    m = 0.f;
    for (int w = 0; w < 16; ++w) m = fmaxf(m, buf[w]);
    sc = pow2_to(__float_as_uint(m), each ? 15 : 14);
    if (!each)
      for (int t = threadIdx.x; t < n; t += 1024) coef[t].x *= sc;   // this thread's own
  }
  if (threadIdx.x != 0) return;
  // (no row counts: 0, whatever the upstream gradient)
  const float f = per_row ? 1.f : n == 0 ? 0.f : dloss[0] * factor * (mean ? 1.f / (float)n : 1.f);
  scale[0] = f / sc, scale[1] = each ? f : f / sc;
}

// The hidden states divided by their rows' powers of two, times dw's (a row a workgroup).
__global__ void __launch_bounds__(256)
scale_h_kernel(State st, const float* __restrict__ unscale, const float* scale, int Dp, f16* __restrict__ out) {
  const int t = blockIdx.x;
  if (t >= st.hdr->n) return;
  const float k = unscale[t] / scale[0];
  const f16* h = reinterpret_cast<const f16*>(st.h) + (int64_t)t * Dp;
  for (int c = threadIdx.x * 8; c < Dp; c += 2048) {
    f16 v[8];
    load8(h, c, Dp, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = rr::from_f32<f16>(rr::to_f32(v[e]) * k);
    rr::u16x8_t q;
    __builtin_memcpy(&q, v, sizeof(q));
    *reinterpret_cast<rr::u16x8_t*>(out + (int64_t)t * Dp + c) = q;
  }
}

// dh^T tiles of one part of the piece: m = channels, n = rows, k = the piece's columns.
struct DhArgs {
  const char* w;         // at the piece's first row
  const char* dz;
  int64_t ldw, ldz, plane_z;
  int V, Tp, ndt, splits, cols;   // V: rows of w from the piece on; cols: the piece's columns to whole k steps
  float* out;            // [splits][Tp][Dt]
  int Dt;
  bool first;
  State st;
};
template <typename C, typename Op, int PZ>
__global__ void __launch_bounds__(C::THREADS, 2)
dh_kernel(DhArgs a) {
  constexpr int BM = C::BM, BN = C::BN;
  using P = Product<Op, BM, BN, C::WM, C::WN, true, false>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  const int n = a.st.hdr->n;
  int dt, tt;
  const int tiles = gridDim.x / a.splits, sp = blockIdx.x / tiles;
  tile_of(blockIdx.x - sp * tiles, a.ndt, tiles / a.ndt, dt, tt);
  const int t0 = tt * BN, d0 = dt * BM;
  if (t0 >= n) return;
  const int steps = a.cols / P::BK;
  const int k0 = (int)((int64_t)steps * sp / a.splits) * P::BK, k1 = (int)((int64_t)steps * (sp + 1) / a.splits) * P::BK;
  typename P::Acc acc;
  const Operand A{a.w + d0 * P::EB, a.ldw, 0, a.V, (int)a.ldw - d0 * P::EB};
  const Operand B{a.dz + (int64_t)t0 * a.ldz, a.ldz, a.plane_z, a.Tp - t0, a.cols * P::EB};
  P::template run<PZ>(acc, A, B, k0, k1, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / P::WN, wn = wave % P::WN;
#pragma unroll
  for (int j = 0; j < P::NI; ++j) {
    const int t = t0 + wn * P::NW + 16 * j + (lane & 15);
    float* o = a.out + ((int64_t)sp * a.Tp + t) * a.Dt + d0 + wm * P::MW + 4 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < P::MI; ++i) {
      float4* at = reinterpret_cast<float4*>(o + 16 * i);
      float4 v = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
      if (!a.first) {
        const float4 u = *at;
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
      }
      *at = v;
    }
  }
}

// A gradient from its parts, in the inputs' type: dh of every row (0 for rows that do not
// count), or dw.  A workgroup per row and 1024 channels, four a thread.
template <typename X, bool DH>
__global__ void __launch_bounds__(256)
sum_out_kernel(State st, const float* __restrict__ part, int D, int64_t ldp, int64_t stride, int splits,
               const float* scale, const float* unscale, X* __restrict__ out) {
  const int64_t row = blockIdx.x;
  const int c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (c >= D) return;
  const int64_t t = DH ? st.pos[row] : row;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (t >= 0) {
    const float f = scale[0] * (unscale != nullptr ? unscale[t] : 1.f);
    const float* at = part + t * ldp + c;   // ldp is whole tiles
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(at + (int64_t)i * stride);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    s.x *= f, s.y *= f, s.z *= f, s.w *= f;
  }
  X* o = out + row * D + c;
  const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < D) o[e] = rr::from_f32<X>(v[e]);
}

// dw^T tiles of the piece: m = channels, n = the piece's columns, k = rows.
struct DwArgs {
  const char* h;
  const char* dz;
  int64_t ldh, ldz, plane_z;
  int V, D, ndt;         // V: rows of dw from the piece on
  const float* scale;
  void* out;             // dw at the piece's first row
  float* part;           // CUT: [cuts][Vp][Dt]
  int64_t ldp, ldcut;
  int cuts;
  State st;
};
template <typename C, typename Op, typename X, int PZ, bool CUT>
__global__ void __launch_bounds__(C::THREADS, 2)
dw_kernel(DwArgs a) {
  constexpr int BM = C::BM, BN = C::BN;
  using P = Product<Op, BM, BN, C::WM, C::WN, true, true>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  const int n = a.st.hdr->n;
  int dt, vt;
  const int tiles = CUT ? gridDim.x / a.cuts : gridDim.x, cut = CUT ? blockIdx.x / tiles : 0;
  tile_of(blockIdx.x - cut * tiles, a.ndt, tiles / a.ndt, dt, vt);
  const int d0 = dt * BM, v0 = vt * BN;
  typename P::Acc acc;
  const Operand A{a.h + d0 * P::EB, a.ldh, 0, n, (int)a.ldh - d0 * P::EB};
  const Operand B{a.dz + (int64_t)v0 * P::EB, a.ldz, a.plane_z, n, BN * P::EB};
  const int steps = (n + P::BK - 1) / P::BK;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / P::WN, wn = wave % P::WN;
  if constexpr (CUT) {
    const int k0 = (int)((int64_t)steps * cut / a.cuts) * P::BK, k1 = (int)((int64_t)steps * (cut + 1) / a.cuts) * P::BK;
    P::template run<PZ>(acc, A, B, k0, k1, lds);
#pragma unroll
    for (int j = 0; j < P::NI; ++j) {
      float* o = a.part + cut * a.ldcut + (int64_t)(v0 + wn * P::NW + 16 * j) * a.ldp + d0 + wm * P::MW;
      store_block<P::MI>(reinterpret_cast<float*>(lds) + wave * 16 * (P::MW + 4), lane, [&](int i) { return acc[i][j]; },
                         [&](int r, int c, f32x4_t x) { *reinterpret_cast<f32x4_t*>(o + (int64_t)r * a.ldp + c) = x; });
    }
    return;
  }
  P::template run<PZ>(acc, A, B, 0, steps * P::BK, lds);
  const float f = a.scale[0];
#pragma unroll
  for (int j = 0; j < P::NI; ++j) {
    using Bits = typename std::conditional<sizeof(X) == 4, float, uint16_t>::type;   // of X
    typedef Bits Four __attribute__((ext_vector_type(4)));
    typedef Bits Vec __attribute__((ext_vector_type(16 / sizeof(X))));
    typedef Vec Any __attribute__((aligned(sizeof(X))));   // rows of dw start at any element
    const int v = v0 + wn * P::NW + 16 * j, d = d0 + wm * P::MW;
    Bits* o = static_cast<Bits*>(a.out) + (int64_t)v * a.D + d;
    store_block<P::MI>(reinterpret_cast<Bits*>(lds) + wave * 16 * (P::MW + 16 / (int)sizeof(X)), lane, [&](int i) {
      Four x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __builtin_bit_cast(Bits, rr::from_f32<X>(acc[i][j][e] * f));
      return x;
    }, [&](int r, int c, Vec x) {
      if (v + r >= a.V) return;
      Bits* at = o + (int64_t)r * a.D + c;
      if (d + c + (int)(16 / sizeof(X)) <= a.D) {
        *reinterpret_cast<Any*>(at) = x;
      } else {
#pragma unroll
        for (int e = 0; e < (int)(16 / sizeof(X)); ++e)
          if (d + c + e < a.D) at[e] = x[e];
      }
    });
  }
}

// ------------------------------------------------------------------ host
int check_dims(const char* who, int64_t T, int64_t D, int64_t V, int64_t K, int dtype, int reduction) {
  const std::string w(who);
  if (T < 0 || D <= 0 || V <= 0) return rr::fail(RR_EINVAL, w + ": rows must be >= 0, channels and vocabulary > 0");
  if (!rr::valid_dtype(dtype)) return rr::fail(RR_EINVAL, w + ": unsupported dtype");
  if (reduction < 0 || reduction > 2) return rr::fail(RR_EINVAL, w + ": reduction must be 0 (none), 1 (mean) or 2 (sum)");
  if (K < 1 || K > kMaxEntries) {
    return rr::fail(RR_EUNSUPPORTED, w + ": 1 to " + std::to_string(kMaxEntries) + " teacher entries a row, got " +
                                         std::to_string(K));
  }
  if (V > kMaxVocab || D > kMaxChannels) {
    return rr::fail(RR_EUNSUPPORTED, w + ": at most " + std::to_string(kMaxVocab) + " words and " +
                                         std::to_string(kMaxChannels) + " channels");
  }
  if (T >= ((int64_t)1 << 24) || up(V, 256) / 256 * (up(T, 64) / 64) >= (1 << 23)) {   // grids below 2^32 threads
    return rr::fail(RR_EUNSUPPORTED, w + ": too many rows");
  }
  return RR_OK;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

LogitArgs logit_args(const Plan& p, const State& st, const void* weight, int K, float tau) {
  LogitArgs a{};
  a.w = p.copy_w ? st.w : static_cast<const char*>(weight);
  a.h = st.h;
  a.ldw = (p.copy_w ? p.Dp : p.D) * p.eb, a.ldh = p.Dp * p.eb;
  a.V = (int)p.V, a.Dp = (int)p.Dp, a.K = K, a.Tp = (int)p.Tp;
  a.c = kLog2e / tau;
  a.st = st;
  return a;
}
// The logits of `cols` columns (whole tiles).
template <typename C, typename Op, Mode MODE, int PZ>
void launch_logits(LogitArgs a, int64_t T, int64_t cols, hipStream_t s) {
  a.nvt = (int)(cols / C::BM);
  logits_kernel<C, Op, MODE, PZ><<<(unsigned)(a.nvt * (up(T, C::BN) / C::BN) * (MODE == kCut ? a.cuts : 1)), C::THREADS, 0, s>>>(a);
}
// The forward's, whole or in parts.
template <typename C, typename Op>
void launch_forward(const LogitArgs& a, const Plan& p, hipStream_t s) {
  if (p.cuts > 1) launch_logits<C, Op, kCut, 1>(a, p.T, p.Vt, s);
  else launch_logits<C, Op, kStats, 1>(a, p.T, p.Vt, s);
}
template <typename C, typename Op, int PZ>
void launch_dh(DhArgs a, const Plan& p, hipStream_t s) {
  a.ndt = (int)(up(p.D, C::BM) / C::BM);
  dh_kernel<C, Op, PZ><<<(unsigned)(a.ndt * (up(p.T, C::BN) / C::BN) * p.splits), C::THREADS, 0, s>>>(a);
}
template <typename C, typename Op, typename X, int PZ, bool CUT>
void launch_dw(DwArgs a, const Plan& p, int64_t cols, hipStream_t s) {
  a.ndt = (int)(up(p.D, C::BM) / C::BM);
  const unsigned tiles = (unsigned)(a.ndt * (cols / C::BN));
  dw_kernel<C, Op, X, PZ, CUT><<<CUT ? tiles * (unsigned)a.cuts : tiles, C::THREADS, 0, s>>>(a);
  if constexpr (CUT) {
    sum_out_kernel<X, false><<<dim3((unsigned)std::min<int64_t>(cols, a.V), (unsigned)((p.D + 1023) / 1024)), 256, 0, s>>>(
        a.st, a.part, a.D, a.ldp, a.ldcut, a.cuts, a.scale, nullptr, static_cast<X*>(a.out));
  }
}

template <typename X, typename Op>
int forward(const Plan& p, const void* hidden, const void* weight, const State& st, const FwdWs& ws, int K, bool labels,
            float zl, float tau, int reduction, float* loss, hipStream_t s) {
  // the weight too where it is not an operand itself
  const int64_t most = p.copy_w ? std::max(p.T, p.V) : p.T;
  pack_kernel<X><<<dim3((unsigned)std::min<int64_t>(8192, most), p.copy_w ? 2 : 1), 256, 0, s>>>(
      static_cast<const X*>(hidden), static_cast<const X*>(weight), p.V, (int)p.D, (int)p.Dp, st);
  LogitArgs a = logit_args(p, st, weight, K, tau);
  a.part = ws.part;
  a.z = p.cuts > 1 ? ws.cut : st.z, a.ldzf = p.Vt, a.ldcut = p.T * p.Vt, a.cuts = (int)p.cuts;
  if (p.rows == kTile32) launch_forward<Tile32, Op>(a, p, s);
  else if (p.rows == kTile64) launch_forward<Tile64, Op>(a, p, s);
  else if constexpr (!__is_same(Op, OpF32)) launch_forward<Tile256, Op>(a, p, s);
  int64_t parts = p.Vt / kEdge;
  if (p.cuts > 1) {
    parts = up(p.Vt, kSeg) / kSeg;
    join_kernel<<<dim3((unsigned)p.T, (unsigned)parts), 256, 0, s>>>(st, ws.cut, a.cuts, a.ldcut, a.V, p.Vt, K, a.c, p.Tp,
                                                                    ws.part);
  }
  float* rows = reduction == 0 ? loss : st.loss;
  row_loss_kernel<<<(unsigned)((p.T + 3) / 4), 256, 0, s>>>(st, ws.part, (int)parts, p.Tp, K, labels, zl, tau, rows);
  if (reduction != 0) sum_loss_kernel<<<1, 1024, 0, s>>>(st.loss, p.T, st.hdr, reduction == 1, loss);
  return rr::check_launch("rr_linear_loss");
}

template <typename X, typename Op, int PZ>
int backward(const Plan& p, const float* dloss, const void* weight, const State& st, const BwdWs& ws, int K, float zl,
             float tau, int reduction, void* dh, void* dw, hipStream_t s) {
  const bool each = __is_same(Op, OpF16) && reduction == 0;   // a power of two for each row's dz
  coef_kernel<<<1, 1024, 0, s>>>(st, dloss, reduction == 0, reduction == 1, tau, zl, __is_same(Op, OpF16), ws.coef,
                                 ws.unscale, ws.scale);
  if (each && dw != nullptr) {
    scale_h_kernel<<<(unsigned)p.T, 256, 0, s>>>(st, ws.unscale, ws.scale, (int)p.Dp, reinterpret_cast<f16*>(ws.h));
  }
  for (int64_t v = 0; v < p.Vt; v += p.Vp) {
    const int64_t cols = std::min(p.Vp, p.Vt - v);   // whole tiles
    LogitArgs a = logit_args(p, st, weight, K, tau);
    a.coef = ws.coef, a.dz = ws.dz, a.ldz = p.Vp * p.eb, a.plane_z = p.Tp * a.ldz, a.v_first = (int)v;
    constexpr bool kFp32 = __is_same(Op, OpF32), kFew = PZ == 2;   // up to kFewRows
    if (kFew || st.z != nullptr) {
      dz_kernel<Op, PZ><<<dim3((unsigned)p.T, (unsigned)(up(cols, kSeg) / kSeg)), 256, 0, s>>>(
          st, ws.coef, a.V, p.Vt, K, a.v_first, (int)cols, ws.dz, a.ldz, a.plane_z);
    } else if constexpr (!kFew) {
      launch_logits<typename std::conditional<kFp32, Tile64, Tile256>::type, Op, kGrad, PZ>(a, p.T, cols, s);
    }
    if (dh != nullptr) {
      DhArgs b{};
      b.w = a.w + v * a.ldw, b.dz = ws.dz, b.ldw = a.ldw, b.ldz = a.ldz, b.plane_z = a.plane_z;
      b.V = (int)(p.V - v), b.Tp = a.Tp, b.splits = (int)p.splits, b.cols = (int)cols;
      b.out = ws.dh, b.Dt = (int)p.Dt, b.first = v == 0, b.st = st;
      if constexpr (kFew || kFp32) {
        if (p.rows == kTile32) launch_dh<Tile32, Op, PZ>(b, p, s);
        else launch_dh<Tile64, Op, PZ>(b, p, s);
      } else {
        launch_dh<Tile256, Op, PZ>(b, p, s);
      }
    }
    if (dw != nullptr) {
      DwArgs c{};
      c.h = each ? ws.h : st.h, c.dz = ws.dz, c.ldh = a.ldh, c.ldz = a.ldz, c.plane_z = a.plane_z;
      c.V = (int)(p.V - v), c.D = (int)p.D, c.scale = ws.scale;
      c.out = static_cast<X*>(dw) + v * p.D, c.st = st;
      c.part = ws.dw, c.ldp = p.Dt, c.ldcut = p.Vp * p.Dt, c.cuts = (int)p.cuts_w;
      if (kFew || p.cuts_w == 1) {
        launch_dw<Tile256, Op, X, PZ, false>(c, p, cols, s);
      } else if constexpr (!kFew) {
        launch_dw<Tile256, Op, X, PZ, true>(c, p, cols, s);
      }
    }
  }
  if (dh != nullptr) {
    sum_out_kernel<X, true><<<dim3((unsigned)p.T, (unsigned)((p.D + 1023) / 1024)), 256, 0, s>>>(
        st, ws.dh, (int)p.D, p.Dt, p.Tp * p.Dt, (int)p.splits, ws.scale + 1, each ? ws.unscale : nullptr, static_cast<X*>(dh));
  }
  return rr::check_launch("rr_linear_loss_bwd");
}

// One more kernel for what has no rows: the loss is 0, the gradients are 0.
__global__ void zero_kernel(uint32_t* p, int64_t words, uint16_t* tail) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) p[i] = 0;
  if (tail != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *tail = 0;
}
void zero(void* p, int64_t bytes, hipStream_t s) {
  if (p == nullptr || bytes == 0) return;
  zero_kernel<<<1024, 256, 0, s>>>(static_cast<uint32_t*>(p), bytes / 4,
                                   bytes % 4 ? static_cast<uint16_t*>(p) + bytes / 2 - 1 : nullptr);
}

int run_forward(const void* hidden, const void* weight, int dtype, int64_t T, int64_t D, int64_t V, int64_t K, bool labels,
                float zl, float tau, int reduction, float* loss, const State& st, void* workspace, hipStream_t s) {
  const Plan p = plan_of(T, D, V, dtype);
  FwdWs ws;
  fwd_layout(p, static_cast<char*>(workspace), &ws);
  if (dtype == RR_BF16) return forward<bf16, OpBf16>(p, hidden, weight, st, ws, (int)K, labels, zl, tau, reduction, loss, s);
  if (dtype == RR_F16) return forward<f16, OpF16>(p, hidden, weight, st, ws, (int)K, labels, zl, tau, reduction, loss, s);
  return forward<float, OpF32>(p, hidden, weight, st, ws, (int)K, labels, zl, tau, reduction, loss, s);
}

int check_buffers(const char* who, int64_t T, int64_t D, int64_t V, int64_t K, int dtype, int pass, const void* hidden,
                  const void* weight, const void* state, size_t state_bytes, const void* ws, size_t ws_bytes) {
  const std::string w(who);
  if ((pass == 0 && hidden == nullptr) || weight == nullptr || state == nullptr || ws == nullptr) return rr::fail(RR_EINVAL, w + ": null pointer");
  if (!aligned16(hidden) || !aligned16(weight)) return rr::fail(RR_EINVAL, w + ": buffers must be 16-byte aligned");
  if (state_bytes < rr_linear_loss_state_bytes(T, D, V, K, dtype, pass == 0 ? 0 : 2)) return rr::fail(RR_EWORKSPACE, w + ": state buffer too small");
  if (ws_bytes < rr_linear_loss_workspace_bytes(T, D, V, dtype, pass)) return rr::fail(RR_EWORKSPACE, w + ": workspace too small");
  if (!aligned16(state) || !aligned16(ws)) return rr::fail(RR_EWORKSPACE, w + ": state buffer or workspace misaligned");
  return RR_OK;
}

// The caller's state: with the logits that it has room for.
void lay_out_state(int64_t T, int64_t D, int64_t V, int64_t K, int dtype, void* state, size_t bytes, State* st) {
  const Plan p = plan_of(T, D, V, dtype);
  const int grad = bytes >= state_layout(p, K, 1, nullptr, nullptr) ? 1 : bytes >= state_layout(p, K, 2, nullptr, nullptr) ? 2 : 0;
  state_layout(p, K, grad, static_cast<char*>(state), st);
}

}  // namespace

extern "C" size_t rr_linear_loss_state_bytes(int64_t rows, int64_t D, int64_t V, int64_t K, int dtype, int grad) {
  if (rows <= 0 || grad < 0 || grad > 2 || check_dims("rr_linear_loss_state_bytes", rows, D, V, K, dtype, 0) != RR_OK) return 0;
  const Plan p = plan_of(rows, D, V, dtype);
  return state_layout(p, K, grad, nullptr, nullptr);
}

extern "C" size_t rr_linear_loss_workspace_bytes(int64_t rows, int64_t D, int64_t V, int dtype, int pass) {
  if (rows <= 0 || check_dims("rr_linear_loss_workspace_bytes", rows, D, V, 1, dtype, 0) != RR_OK) return 0;
  const Plan p = plan_of(rows, D, V, dtype);
  return pass == 0 ? fwd_layout(p, nullptr, nullptr) : bwd_layout(p, nullptr, nullptr);
}

extern "C" int rr_linear_ce_fwd(const void* hidden, const void* weight, int dtype, int64_t rows, int64_t D, int64_t V,
                                const int64_t* labels, int64_t ignore_index, float z_loss, int reduction, float* loss,
                                void* state, size_t state_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "rr_linear_ce_fwd";
  if (int rc = check_dims(who, rows, D, V, 1, dtype, reduction)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows > 0 || reduction != 0) {
    if (loss == nullptr) return rr::fail(RR_EINVAL, std::string(who) + ": null pointer");
  }
  if (rows == 0) {
    if (reduction != 0) zero(loss, 4, s);
    return rr::check_launch(who);
  }
  if (labels == nullptr) return rr::fail(RR_EINVAL, std::string(who) + ": null pointer");
  if (int rc = check_buffers(who, rows, D, V, 1, dtype, 0, hidden, weight, state, state_bytes, workspace, workspace_bytes)) return rc;
  State st;
  lay_out_state(rows, D, V, 1, dtype, state, state_bytes, &st);
  State in = st;
  if (reduction == 0) in.loss = loss;   // where rows that do not count leave their 0
  rows_kernel<true><<<1, 1024, 0, s>>>(labels, ignore_index, rows, (int)V, in);
  return run_forward(hidden, weight, dtype, rows, D, V, 1, true, z_loss, 1.f, reduction, loss, st, workspace, s);
}

extern "C" int rr_linear_kd_fwd(const void* hidden, const void* weight, int dtype, int64_t rows, int64_t D, int64_t V,
                                const void* teacher_logits, int teacher_dtype, const int64_t* teacher_ids, int64_t K,
                                float temperature, int reduction, float* loss, void* state, size_t state_bytes,
                                void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "rr_linear_kd_fwd";
  if (int rc = check_dims(who, rows, D, V, K, dtype, reduction)) return rc;
  if (!rr::valid_dtype(teacher_dtype)) return rr::fail(RR_EINVAL, std::string(who) + ": unsupported teacher dtype");
  if (!(temperature > 0.f) || !(temperature < 1e30f)) {
    return rr::fail(RR_EINVAL, std::string(who) + ": temperature must be positive and finite");
  }
  if (rows * K >= ((int64_t)1 << 31)) return rr::fail(RR_EUNSUPPORTED, std::string(who) + ": too many teacher entries");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows > 0 || reduction != 0) {
    if (loss == nullptr) return rr::fail(RR_EINVAL, std::string(who) + ": null pointer");
  }
  if (rows == 0) {
    if (reduction != 0) zero(loss, 4, s);
    return rr::check_launch(who);
  }
  if (teacher_logits == nullptr || teacher_ids == nullptr) return rr::fail(RR_EINVAL, std::string(who) + ": null pointer");
  if (int rc = check_buffers(who, rows, D, V, K, dtype, 0, hidden, weight, state, state_bytes, workspace, workspace_bytes)) return rc;
  State st;
  lay_out_state(rows, D, V, K, dtype, state, state_bytes, &st);
  int KP = 1;
  while (KP < K) KP *= 2;
  RR_DISPATCH_DTYPE(teacher_dtype, {
    entries_kernel<InT><<<(unsigned)rows, 64, (size_t)KP * 8, s>>>(static_cast<const InT*>(teacher_logits), teacher_ids, (int)K,
                                                                  KP, (int)V, temperature, st.ids, st.p, st.pos);
  });
  State in = st;
  if (reduction == 0) in.loss = loss;
  rows_kernel<false><<<1, 1024, 0, s>>>(nullptr, 0, rows, (int)V, in);
  return run_forward(hidden, weight, dtype, rows, D, V, K, false, 0.f, temperature, reduction, loss, st, workspace, s);
}

extern "C" int rr_linear_loss_bwd(const float* dloss, const void* weight, int dtype, int64_t rows, int64_t D,
                                  int64_t V, int64_t K, float z_loss, float temperature, int reduction,
                                  const void* state, size_t state_bytes, void* dhidden, void* dweight, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const char* who = "rr_linear_loss_bwd";
  if (int rc = check_dims(who, rows, D, V, K, dtype, reduction)) return rc;
  if (!(temperature > 0.f) || !(temperature < 1e30f)) {
    return rr::fail(RR_EINVAL, std::string(who) + ": temperature must be positive and finite");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t es = dtype == RR_F32 ? 4 : 2;
  if (rows == 0) {
    zero(dweight, V * D * es, s);
    return rr::check_launch(who);
  }
  if (dloss == nullptr) return rr::fail(RR_EINVAL, std::string(who) + ": null pointer");
  if (int rc = check_buffers(who, rows, D, V, K, dtype, 1, nullptr, weight, state, state_bytes, workspace, workspace_bytes)) return rc;
  if (dhidden == nullptr && dweight == nullptr) return RR_OK;
  const Plan p = plan_of(rows, D, V, dtype);
  State st;
  lay_out_state(rows, D, V, K, dtype, const_cast<void*>(state), state_bytes, &st);
  BwdWs ws;
  bwd_layout(p, static_cast<char*>(workspace), &ws);
#define LL_BACKWARD(X, OP, PZ) \
  backward<X, OP, PZ>(p, dloss, weight, st, ws, (int)K, z_loss, temperature, reduction, dhidden, dweight, s)
  if (dtype == RR_BF16) return p.planes_z == 2 ? LL_BACKWARD(bf16, OpBf16, 2) : LL_BACKWARD(bf16, OpBf16, 1);
  if (dtype == RR_F16) return p.planes_z == 2 ? LL_BACKWARD(f16, OpF16, 2) : LL_BACKWARD(f16, OpF16, 1);
  return LL_BACKWARD(float, OpF32, 1);
#undef LL_BACKWARD
}
