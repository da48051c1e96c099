// linear_loss.hip — losses over a large vocabulary straight from hidden states, on
// gfx950: cross entropy on labels, distillation from a teacher's top logits, and the
// losses on the labels' log-probabilities.
//
//   z = h w^T  [rows, V];  s = z / tau;  lse = log sum_v exp(s_v);  q = exp(s - lse)
//   cross entropy (tau = 1)  loss = lse - z_label + zl lse^2
//                            dz = c ((1 + 2 zl lse) q - 1[v = label])
//   distillation             p = softmax over the row's teacher entries of t / tau
//                            loss = tau^2 sum_k p_k (log p_k - log q_{id_k})
//                            dz = c tau (q - sum_{k: id_k = v} p_k)
//   dh = dz w,  dw = dz^T h,  c the row's upstream gradient
//
//   log-probabilities        logp = s_label - lse;  dz = c / tau (1[v = label] - q)
//   clipped policy           r = exp(logp - old), d = ref - logp
//                            loss = -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl (exp(d) - d - 1)
//                            c = -[r not clipped] r A + kl (1 - exp(d))
//   preference               S = sum of a sequence's logp, m = beta ((S_1 - ref_1) - (S_2 - ref_2)) of a pair
//                            loss = -(1 - eps) log sigmoid(m) - eps log sigmoid(-m)
//                            c = +- beta (eps sigmoid(m) - (1 - eps) sigmoid(-m)) for all tokens of a sequence
//
// A label is a teacher with one entry of weight 1, so all run on the same
// kernels; what the last two put on a log-probability is left by the forward, a value a
// row.  The forward forms the logits a tile at a time and keeps each row's running
// maximum and sum per tile and the logits of the row's entries; where that pays
// (kKeepBytes and kKeepChannels below) and the caller has room it also leaves the logits
// themselves, in fp32.
// The backward reads them, or forms them again, a piece of the vocabulary at a time,
// rounds that piece of dz to the operands' 16 bits (for few rows to two planes of them;
// fp32 inputs: not at all), and uses it for dw (complete for the piece) and dh (added
// up over the pieces in fp32).
//
// What bounds it: with many rows the products, two to four of 2 rows V D flops (8192 x
// 65536 x 2560 bf16 forward and backward 7.3 to 7.5 ms, 1.1 PFLOP/s of the three it cannot do
// without; a large product alone runs at 1.4); with few rows the weight's bytes, read
// once forward and once backward and dw's written (16 x 65536 x 5120 bf16 forward 137 us, 4.9
// TB/s, with the backward 540 us, 3.7 TB/s); below about 200 us the launches, 10 to 15.
// Where a product has fewer tiles than CUs its sum is cut in parts that are joined by a
// launch more (best_parts): the logits' over the channels, dh's over the words, dw's over the
// rows (fp32, 209 rows of 3456 channels, 832 words, forward and backward: 117 us, 3.6 times that whole).
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
// at the end, and dw reads the hidden states divided by it (a copy, for dw sums over rows), where a
// row whose |factor hidden| is below 2^-29 of the largest loses bits, and all of them below 2^-40.
//
// dz of 16-bit inputs is in 16 bits, as they are: with more than kFewRows rows in one plane, which is
// the second rounding of a gradient whose output is the first.  A second plane would undo it at the
// price of twice the products of dw and dh: gradients 2.3e-3 and 1.66e-3 off in the 2-norm, 6.8 and
// 10.9 ms (policy loss, 8192 x 65536 x 2560 bf16), 133 and 179 us (preference loss, 512 x 32000 x 768).
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
// x 2560 7.5 and 9.0 ms.  fp32 products cost more, so theirs are kept from a twelfth of the
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
// the loads, and small tiles fill the last round (with Tile256 300 x 5003 x 1000 forward and
// backward took 29 % longer, 2048 x 32000 x 2048 1.5 % less).
struct Tile256 { static constexpr int BM = 256, BN = 256, WM = 2, WN = 4, THREADS = 512; };
struct Tile64 { static constexpr int BM = 256, BN = 64, WM = 4, WN = 1, THREADS = 256; };
struct Tile32 { static constexpr int BM = 256, BN = 32, WM = 4, WN = 1, THREADS = 256; };
// Half of a Tile256, for the last round of tiles where that leaves half of the CUs or more without
// work: then two workgroups take a tile's halves (half_work), in about 0.8 of a round where it has 12 or 18 steps
// (1152 rows of 768 channels and 32000 words: logits 76.5 and 72.8 us, dw 64.0 and 60.9).
struct Half256 { static constexpr int BM = 256, BN = 128, WM = 2, WN = 4, THREADS = 512; };
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
  int count;             // what the mean is over: those rows, or the pairs that count
  float top;             // the largest of the rows' derivatives that the forward left (State.z2)
  int whole, parts;      // the losses on log-probabilities: DhShare
};
struct State {
  Header* hdr;
  int* rows;     // [rows] the i-th row that counts
  int* pos;      // [rows] its place there, -1 for a row that does not count
  float* lse2;   // [rows] log2 of the row's sum of exponentials (in the order of `rows`)
  float* loss;   // [rows]
  int* ids;      // [rows][K] the entries' columns, ascending; kAbsent past the last
  float* p;      // [rows][K] their weights
  float* z2;     // [rows][K] their logits, times log2(e) / tau; the policy and the preference loss leave
                 // the derivative of a row's loss by -logp there instead, for the backward
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
  bool small_w;        // fp32 losses on log-probabilities: dw whole on Tile64 in place of parts on Tile256
};
constexpr int64_t kCus = 256;
// Seconds of a k step of a round of tiles, against which the parts' bytes (at 4 TB/s, written and read)
// and a launch are weighed: with fp32's at 1.4 us too 300 x 5003 x 1000 forward and backward took 14 %
// longer, 4678 x 30720 x 535 10 % (but 512 x 32000 x 768 3.5 % less).
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
    // fp32: small tiles, which are half a Tile256's k step for a quarter of its work, fill the GPU without parts
    // (dw of 460 rows, 512 channels, 16001 words: 95 us in two parts, 71 so).
    const int64_t tiles = p.Dt / kEdge * (p.Vp / kEdge);
    const double whole = (double)((4 * tiles + 2 * kCus - 1) / (2 * kCus)) * (double)steps * kStepF32;
    const double parts = (double)((tiles * p.cuts_w + kCus - 1) / kCus) * (double)steps / (double)p.cuts_w * kStepF32Dw +
                         (p.cuts_w > 1 ? (double)(p.cuts_w * p.Vp * D * 8) / 4e12 + kLaunch : 0.);
    p.small_w = p.fp32 && whole < parts;
  }
  return p;
}

// Whether the logits that are kept are more than the 256 MB cache holds: they are then written past it
// (6.6 x 10^3 and 7.4 x 10^3 rows of 65536 bf16: the forward's product 2030 and 2272 us, 1840 and 2055 so).
bool keeps_past(const Plan& p) { return p.T * p.Vt * 4 > (int64_t)256 << 20; }

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
  float* scale;    // the factors on dw and on dh, and dw's power of two
  float2* coef;    // [Tp] a row's factors (coef_kernel)
  float* unscale;  // [Tp] the inverse of a row's power of two (fp16)
  char* h;         // [T][Dp] the hidden states times that (fp16)
  char* dz;        // [planes_z][Tp][Vp]
  float* dh;       // [splits][Tp][Dt]; log-probabilities: [Tp][Dt], then the shared tiles' parts (DhShare)
  float* dw;       // [cuts_w][Vp][Dt], where there are two or more and they are used
};
// dh's tiles in the losses on log-probabilities.  How many rows count is known on the device
// alone, and with it how many tiles there are: as many as fill whole rounds of the GPU are done by a
// workgroup each, the others are shared by `parts` workgroups each, along the vocabulary.  Cut in
// as many equal parts as suit all rows (best_parts), 26 x 10 tiles of 32 x 10 took four rounds of a third
// each: 1117 us where they take 900 (8192 rows, a fifth ignored, 2560 channels, 32768 words bf16).
struct DhShare {
  int whole, parts;
};
struct DhShape {
  int ndt, bn;       // tiles of channels, rows of a tile
  int slots;         // workgroups at one time
  int room;          // parts that there is room for
  int steps;         // of k in a piece
  float cost;        // of a part's writing and reading, in steps
};
// (by a wave: a lane tries a number of parts)
__device__ __forceinline__ DhShare dh_share(const DhShape& a, int n, int lane) {
  const int tiles = a.ndt * ((n + a.bn - 1) / a.bn), rest = tiles % a.slots;
  int s = lane + 1;
  float c = (float)((rest * s + a.slots - 1) / a.slots * a.steps) / (float)s + (float)(s * rest) * a.cost;
  if (s > 1 && (rest * s > a.room || 4 * s > a.steps)) c = INFINITY;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float c2 = __shfl_xor(c, o, 64);
    const int s2 = __shfl_xor(s, o, 64);
    if (c2 < c || (c2 == c && s2 < s)) c = c2, s = s2;
  }
  return {tiles - rest, s};
}
DhShape dh_shape(const Plan& p) {
  const bool big = p.rows == kTile256;
  DhShape a;
  a.bn = big ? Tile256::BN : p.rows == kTile64 ? Tile64::BN : Tile32::BN;
  a.ndt = (int)(p.Dt / kEdge), a.slots = (int)(big ? kCus : 2 * kCus);
  const int64_t tiles = up(p.T, a.bn) / a.bn * a.ndt;
  a.room = (int)std::min<int64_t>(2 * a.slots, 64 * tiles);
  a.steps = (int)(p.Vp * p.eb / 128) * p.planes_z;
  a.cost = (float)((double)(kEdge * a.bn * 8) / 4e12 / (p.fp32 ? kStepF32 : kStep));
  return a;
}
size_t dh_bytes(const Plan& p, bool logp) {
  if (!logp) return (size_t)p.splits * p.Tp * p.Dt * 4;
  const DhShape a = dh_shape(p);
  return (size_t)(p.Tp * p.Dt + (int64_t)a.room * kEdge * a.bn) * 4;
}
size_t bwd_layout(const Plan& p, bool logp, char* base, BwdWs* s) {
  Carve take{base};
  BwdWs t;
  t.scale = reinterpret_cast<float*>(take(256));
  t.coef = reinterpret_cast<float2*>(take((size_t)p.Tp * sizeof(float2)));
  t.unscale = reinterpret_cast<float*>(take(p.dtype == RR_F16 ? (size_t)p.Tp * 4 : 0));
  t.h = take(p.dtype == RR_F16 ? (size_t)p.T * p.Dp * p.eb : 0);
  t.dz = take((size_t)p.planes_z * p.Tp * p.Vp * p.eb);
  t.dh = reinterpret_cast<float*>(take(dh_bytes(p, logp)));
  t.dw = reinterpret_cast<float*>(take(p.cuts_w > 1 && !(logp && p.small_w) ? (size_t)p.cuts_w * p.Vp * p.Dt * 4 : 0));
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
  if (tid == 0) st.hdr->n = base, st.hdr->count = base;
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

// A row of an operand by a workgroup: copied, padded with zeros to Dp channels.  amax: null, or where
// fp16's largest finite |value| goes.
template <typename X>
__device__ __forceinline__ void pack_row(const X* xr, int D, int Dp, X* out, float* amax, float* buf) {
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
    *reinterpret_cast<Words*>(out + c) = q;
  }
  if constexpr (__is_same(X, f16)) {
    if (amax == nullptr) return;
    m = wave_max(m);
    __syncthreads();   // the last row's reads of buf are done
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) *amax = fmaxf(fmaxf(buf[0], buf[1]), fmaxf(buf[2], buf[3]));
  }
}

// rows_kernel<true> and pack_kernel in one launch, for few rows: a workgroup a row, which
// finds its place by reading the labels in front of it (1536 rows of 768 channels: 9.7 us in two
// launches, 5.3 in one; with 2048 rows that is 16 MB from the caches).
constexpr int64_t kRowsInOne = 2048;
template <typename X>
__global__ void __launch_bounds__(256)
rows_pack_kernel(const X* __restrict__ hidden, const X* __restrict__ weight, const int64_t* __restrict__ labels,
                 int64_t ignore, int T, int V, int D, int Dp, State st, float* __restrict__ loss) {
  __shared__ float buf[4];
  __shared__ int counts[4];
  const int tid = threadIdx.x;
  if (blockIdx.y == 1) {
    for (int64_t r = blockIdx.x; r < V; r += gridDim.x) pack_row(weight + r * D, D, Dp, reinterpret_cast<X*>(st.w) + r * Dp, nullptr, buf);
    return;
  }
  const int row = blockIdx.x;
  if (row >= T) return;
  int before = 0;
  for (int i = tid; i < row; i += 256) before += labels[i] != ignore ? 1 : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
  if ((tid & 63) == 0) counts[tid >> 6] = before;
  __syncthreads();
  const int at = (counts[0] + counts[1]) + (counts[2] + counts[3]);
  const int64_t l = labels[row];
  const bool in = l != ignore;
  if (tid == 0) {
    const bool ok = l >= 0 && l < V;
    st.ids[row] = ok ? (int)l : kAbsent;
    st.p[row] = ok || !in ? 1.f : NAN;
    st.pos[row] = in ? at : -1;
    if (in) st.rows[at] = row;
    if (!in) loss[row] = 0.f;
    if (row == T - 1) st.hdr->n = st.hdr->count = at + (in ? 1 : 0);
  }
  if (in) pack_row(hidden + (int64_t)row * D, D, Dp, reinterpret_cast<X*>(st.h) + (int64_t)at * Dp, st.amax + at, buf);
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
    pack_row(xr, D, Dp, out + r * Dp, w ? nullptr : st.amax + r, buf);
  }
}

// What multiplies a row of dz where nothing has to be known of the other rows (the losses on
// log-probabilities in bf16 and fp32): found where dz is made, coef_kernel's launch saved (2.4 us of 146
// for 512 rows of 768 channels and 32000 words, 8 of 6300 for 8192).
//
// All tokens of a sequence may share one factor c, and -c at their words is off by the same rounding in
// all of them, up to half a step of dz's 16 bits: bf16 gradients are 1.9e-3 to 2.4e-3 off in the 2-norm
// where the mean cross entropy's, whose rows have the factor 1, are 1.9e-3, 4.3e-3 at worst.  (c kept out
// of dz, on dh's rows and on a copy of the hidden states for dw: dh 1.9e-3 and dw 2.6e-3, and 0.5 to 2 %
// more time.)  The largest |c| goes into the factors on dw and dh, so that it is 1 in dz: a single
// pair, or advantages of one size, are off by no more than cross entropy.
struct Upstream {
  const float* dloss;   // [losses], or one for all
  float factor;
  int group;            // rows of a loss
  bool per_row, mean, weighted;
  float* scale;         // the factors on dw and on dh
};
__device__ __forceinline__ float row_factor(const Upstream& u, const State& st, int row) {
  const float c = u.per_row ? u.dloss[u.group == 1 ? row : row / u.group] * u.factor : 1.f;
  return u.weighted ? (u.per_row ? c * st.z2[row] : st.z2[row] / st.hdr->top) : c;
}
__device__ __forceinline__ void leave_scale(const Upstream& u, const State& st) {
  float f = 1.f;   // (no row counts: 0, whatever the upstream gradient)
  if (!u.per_row) f = st.hdr->n == 0 ? 0.f : u.dloss[0] * u.factor * (u.mean ? 1.f / (float)st.hdr->count : 1.f) * st.hdr->top;
  u.scale[0] = f, u.scale[1] = f;
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
  bool past;              // the logits are written past the cache, which would not hold them
  int cuts;
  const float2* coef;     // backward: of coef_kernel, or null
  Upstream up;
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
// Keeps a store past the cache apart from the ordinary one of the other branch: made one, they are ordinary.
__device__ __forceinline__ void apart() { asm volatile(""); }
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

// The workgroup's tile of `tiles` (its number in the order of tile_of's bands) and half: -1 for a
// whole one, 0 or 1 in a last round of halves.  False: it has none.  (kHalfMore workgroups more than tiles.)
constexpr int kHalfMore = (int)kCus / 2;
__device__ __forceinline__ bool half_work(int tiles, int b, int& id, int& half) {
  const int rest = tiles % (int)kCus, whole = tiles - rest;
  half = -1;
  if (2 * rest > (int)kCus) {
    if (b >= tiles) return false;
    id = xcd_order(b, tiles);
  } else if (b < whole) {
    id = xcd_order(b, whole);
  } else {
    if (b - whole >= 2 * rest) return false;
    const int at = xcd_order(b - whole, 2 * rest);
    id = whole + at / 2, half = at & 1;
  }
  return true;
}

// z^T tiles: m = vocabulary, n = rows, so that a lane holds 4 MI logits of a row.
// kStats: the forward's maxima and sums, and the logits where they are kept; kCut: one part of
// the sums, as it is; kGrad: the backward's dz.
enum Mode { kStats, kCut, kGrad };
template <typename C, typename Op, Mode MODE, int PZ>
__device__ __forceinline__ void logits_tile(const LogitArgs& a, char* lds, int n, int vt, int t0, int cut, int k0, int k1) {
  constexpr bool GRAD = MODE == kGrad;
  constexpr int BM = C::BM, BN = C::BN;
  using P = Product<Op, BM, BN, C::WM, C::WN, false, false>;
  const int v0 = a.v_first + vt * BM;
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
      if constexpr (GRAD) {
        co[j] = a.coef != nullptr ? a.coef[t] : make_float2(row_factor(a.up, a.st, orig[j]), 0.f);   // (K is 1)
        l2[j] = a.st.lse2[t];
      }
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
      if (t + r >= n) return;
      f32x4_t* at = reinterpret_cast<f32x4_t*>(o + (int64_t)r * a.ldzf + v);
      if (MODE == kStats && a.past) {
        apart();
        __builtin_nontemporal_store(x, at);
        apart();
      } else {
        *at = x;
      }
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

template <typename C, typename Op, Mode MODE, int PZ>
__global__ void __launch_bounds__(C::THREADS, 2)
logits_kernel(LogitArgs a) {
  constexpr int BN = C::BN;
  constexpr bool kHalves = __is_same(C, Tile256) && MODE != kCut;
  using P = Product<Op, C::BM, BN, C::WM, C::WN, false, false>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  const int n = a.st.hdr->n;
  if constexpr (MODE == kGrad) {
    if (a.coef == nullptr && blockIdx.x == 0 && threadIdx.x == 0) leave_scale(a.up, a.st);
  }
  int vt, tt, id = blockIdx.x, half = -1;
  int k0 = 0, k1 = a.Dp, cut = 0;
  if constexpr (MODE == kCut) {
    const int tiles = gridDim.x / a.cuts, steps = a.Dp / P::BK;
    cut = id / tiles, id -= cut * tiles;
    k0 = steps * cut / a.cuts * P::BK, k1 = steps * (cut + 1) / a.cuts * P::BK;
  }
  // The tiles of the rows that count are dealt out, not of all rows: an XCD takes neighbours,
  // and those of the last rows would leave it without work.
  const int row_tiles = (n + BN - 1) / BN, tiles = a.nvt * row_tiles;
  if constexpr (kHalves) {
    if (!half_work(tiles, blockIdx.x, id, half)) return;
    band_tile(id, a.nvt, row_tiles, vt, tt);
  } else {
    if (id >= tiles) return;
    tile_of(id, a.nvt, row_tiles, vt, tt);
  }
  if constexpr (kHalves) {
    if (half >= 0) {
      const int t0 = tt * BN + half * Half256::BN;
      if (t0 < n) logits_tile<Half256, Op, MODE, PZ>(a, lds, n, vt, t0, cut, k0, k1);
      return;
    }
  }
  logits_tile<C, Op, MODE, PZ>(a, lds, n, vt, tt * BN, cut, k0, k1);
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
dz_kernel(State st, const float2* __restrict__ coef, Upstream up, int V, int64_t Vt, int K, int v_first, int cols,
          char* __restrict__ dz, int64_t ldz, int64_t plane_z) {
  const int t = blockIdx.x;
  if (coef == nullptr && t == 0 && blockIdx.y == 0 && threadIdx.x == 0) leave_scale(up, st);
  if (t >= st.hdr->n) return;
  const int tid = threadIdx.x, rel0 = blockIdx.y * kSeg, at = rel0 + tid * 8, v0 = v_first + rel0, v = v0 + tid * 8;
  const bool here = at < cols;   // both multiples of 8
  const float2 co = coef != nullptr ? coef[t] : make_float2(row_factor(up, st, st.rows[t]), 0.f);
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

// What a policy's loss reads of each row.
struct Policy {
  const float* advantages;   // [rows / per]
  int64_t per;
  const float* old;          // [rows]; null: the log-probabilities of this call
  const float* ref;          // [rows], where kl is not 0
  float lo, hi, kl;          // borders of the ratio, weight of the KL term
};

// exp(d) - d - 1, which is d^2 / 2 and more: close to 0 from its series (below 1/4 its next term is
// 1e-8 of it), where the difference would leave few bits.
__device__ __forceinline__ float exp_rest(float d) {
  if (fabsf(d) < 0.25f)
    return 0.5f * d * d * (1.f + d * (1.f / 3) * (1.f + d * (1.f / 4) * (1.f + d * (1.f / 5) * (1.f + d * (1.f / 6) * (1.f + d * (1.f / 7))))));
  return d > 60.f ? expm1f(d) : expm1f(d) - d;   // (not inf - inf)
}

// Per row: the tiles' maxima and sums to the row's lse and its label's log-probability, to
// `out`; or, POLICY, its loss, and the derivative by -logp for the backward.  A ratio on a border
// of the clipping counts as inside it; without an advantage the ratio counts for nothing,
// however large.  A workgroup takes 16 rows, 16 threads each, so that a wave's loads are whole
// lines (8192 rows of 256 tiles: 16.4 us a wave a row, 10.3 so; 1152 of 125: 5.6 and 5.0).
constexpr int kLogpRows = 16;
template <bool POLICY>
__global__ void __launch_bounds__(256)
row_logp_kernel(State st, const float2* __restrict__ part, int nvt, int64_t Tp, Policy a, DhShape shape, float* __restrict__ out) {
  __shared__ float2 buf[4][kLogpRows];
  const int n = st.hdr->n, t0 = (int)blockIdx.x * kLogpRows;
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x >= 192) {   // for the backward
    const DhShare sh = dh_share(shape, n, threadIdx.x & 63);
    if (threadIdx.x == 192) st.hdr->whole = sh.whole, st.hdr->parts = sh.parts;
  }
  if (t0 >= n) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, mine = threadIdx.x & (kLogpRows - 1);
  const int t = t0 + mine;
  float m = -INFINITY, s = 0.f;
  auto part_of = [](float m2, float s2, float mm) { return m2 == mm ? s2 : s2 * exp2_fast(m2 - mm); };   // (not inf - inf)
  auto join = [&](float m2, float s2) {
    const float mm = fmaxf(m, m2);
    s = part_of(m, s, mm) + part_of(m2, s2, mm);
    m = mm;
  };
  // eight tiles at a time: their loads, their exponentials
  const float2* at = part + (t < n ? t : t0);
  for (int v0 = threadIdx.x / kLogpRows; v0 < nvt; v0 += 128) {
    float2 x[8];
    float mm = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v0 + 16 * i < nvt ? at[(int64_t)(v0 + 16 * i) * Tp] : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) mm = fmaxf(mm, x[i].x);
    s = part_of(m, s, mm), m = mm;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += part_of(x[i].x, x[i].y, mm);
  }
#pragma unroll
  for (int o = kLogpRows; o < 64; o *= 2) join(__shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
  if (lane < kLogpRows) buf[wave][lane] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x >= kLogpRows || t >= n) return;
  m = buf[0][mine].x, s = buf[0][mine].y;
  for (int w = 1; w < 4; ++w) join(buf[w][mine].x, buf[w][mine].y);
  const int64_t row = st.rows[t];
  const float log2s = log2f(s);
  // (the maximum goes first: what is left is small and keeps its bits)
  const float logp = st.ids[row] == kAbsent ? NAN : ((st.z2[row] - m) - log2s) * kLn2;
  float value = logp;
  if constexpr (POLICY) {
    const float A = a.advantages[row / a.per];
    const float r = a.old == nullptr ? (logp != logp ? logp : 1.f) : expf(logp - a.old[row]);
    float by = 0.f;   // by logp
    if (A == 0.f) {
      value = r != r ? r : 0.f;
    } else {
      const bool clipped = A > 0.f ? r > a.hi : r < a.lo;
      value = -(clipped ? (A > 0.f ? a.hi : a.lo) : r) * A;
      by = clipped ? 0.f : value;
    }
    if (a.kl != 0.f) {
      const float d = a.ref[row] - logp;
      value += a.kl * exp_rest(d);
      by -= a.kl * expm1f(d);
    }
    st.z2[row] = -by;
  }
  out[row] = value;
  st.lse2[t] = value != value ? NAN : m + log2s;   // the backward's row is NaN where the loss is
}

// A pair's loss from its sequences' sums, and its derivative by -logp of a token of the first.  In 64
// bits, as the sums are: a sequence's is in the thousands where the difference of two of them decides.
struct Preference {
  const float* ref;   // [pairs][2], or null
  int64_t L;          // tokens of a sequence
  double beta, eps;
};
__device__ __forceinline__ float pair_loss(const Preference& a, double m, int64_t pair, float& by) {
  if (a.ref != nullptr) m -= (double)a.ref[2 * pair] - (double)a.ref[2 * pair + 1];
  m *= a.beta;
  const double e = exp(-fabs(m)), rest = log1p(e);   // -log sigmoid(m) = max(-m, 0) + rest
  const double up = 1 / (1 + e), down = e / (1 + e);   // sigmoid(|m|), sigmoid(-|m|)
  double loss = (1 - a.eps) * (fmax(-m, 0.) + rest);
  if (a.eps != 0) loss += a.eps * (fmax(m, 0.) + rest);   // (not 0 x inf)
  by = (float)(a.beta * (m < 0 ? (1 - a.eps) * up - a.eps * down : (1 - a.eps) * down - a.eps * up));
  return (float)loss;
}

// Of a whole workgroup, what the losses are closed by: their sum, how many count, the largest
// |derivative|; to its first thread.
struct Close {
  float sum, top;
  int count;
};
template <int WAVES>
__device__ __forceinline__ Close close_up(Close c) {
  __shared__ Close buf[WAVES];
  c.sum = wave_add(c.sum), c.top = wave_max(c.top);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c.count += __shfl_xor(c.count, o, 64);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = c;
  __syncthreads();
  Close all{0.f, 0.f, 0};
  for (int w = 0; w < WAVES; ++w) all.sum += buf[w].sum, all.top = fmaxf(all.top, buf[w].top), all.count += buf[w].count;
  return all;
}
// (1 in place of a top whose inverse is no normal value, or before which the other rows' factors would vanish)
__device__ __forceinline__ float usable(float top) { return top > 0x1p-100f && top < 0x1p60f ? top : 1.f; }
__device__ __forceinline__ float finite_abs(float v) { return fabsf(v) < INFINITY ? fabsf(v) : 0.f; }

// The losses of the pairs from their tokens' log-probabilities in st.loss, and their derivative
// by each token's -logp.  A pair without a token that counts counts for nothing.  One launch for few
// tokens: `waves` of the workgroup's 16 take a pair, half of them a sequence (512 tokens: 7.1 us in
// two launches, 6.2 in one; 8192: 11.5 and 13.9).  each: null, or where the pairs' losses go;
// out: null, or where their sum or mean does.
constexpr int64_t kTokensInOne = 2048;
__global__ void __launch_bounds__(1024)
pairs_kernel(State st, Preference a, int64_t pairs, int waves, bool mean, float* __restrict__ each, float* __restrict__ out) {
  __shared__ double sum[16];
  __shared__ int any[16];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int at_once = 16 / waves, half = waves * 32;   // threads of a sequence
  const int mine = tid / (2 * half), k = tid % half, side = tid / half & 1;
  Close c{0.f, 0.f, 0};
  for (int64_t p0 = 0; p0 < pairs; p0 += at_once) {
    const int64_t pair = p0 + mine, first = (pair * 2 + side) * a.L;
    double s = 0;
    int n = 0;
    if (pair < pairs) {
      for (int64_t i = k; i < a.L; i += half) {
        if (st.pos[first + i] < 0) continue;
        s += (double)st.loss[first + i], n = 1;
      }
    }
    // a wave is of one sequence, or, where it has a pair, its halves are
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor(s, o, 64), n |= __shfl_xor(n, o, 64);
    n |= __shfl_xor(n, 32, 64);
    const double other = __shfl_xor(s, 32, 64);
    const double both = waves == 1 ? ((tid & 32) == 0 ? s - other : other - s) : s + other;
    __syncthreads();   // the last turn's reads are done
    if ((tid & 63) == 0) sum[wave] = both, any[wave] = n;
    __syncthreads();
    if (pair >= pairs) continue;
    double m = 0;
    int counts = 0;
    for (int w = 0; w < waves; ++w) {
      const double v = sum[mine * waves + w];
      m += waves == 1 || w < waves / 2 ? v : -v;
      counts |= any[mine * waves + w];
    }
    float by = 0.f;
    const float loss = counts ? pair_loss(a, m, pair, by) : 0.f;
    if (tid % (2 * half) == 0) {
      if (each != nullptr) each[pair] = loss;
      c.sum += loss, c.count += counts, c.top = fmaxf(c.top, finite_abs(by));
    }
    if (!counts) continue;
    for (int64_t i = k; i < a.L; i += half) st.z2[first + i] = side == 0 ? by : -by;
  }
  if (out == nullptr) return;
  c = close_up<16>(c);
  if (tid != 0) return;
  st.hdr->count = c.count, st.hdr->top = usable(c.top);
  out[0] = mean ? c.sum / (float)max(1, c.count) : c.sum;
}

// The same for many tokens, a workgroup a pair.  counted and bys: null, or whether each counts and its |derivative|.
__global__ void __launch_bounds__(256)
pair_kernel(State st, Preference a, float* __restrict__ each, int* __restrict__ counted, float* __restrict__ bys) {
  __shared__ double sum[4];
  __shared__ int any[4];
  const int64_t pair = blockIdx.x;
  const int tid = threadIdx.x, side = tid >> 7;   // half of the threads take one sequence, half the other
  const int64_t first = (pair * 2 + side) * a.L;
  double s = 0;
  int n = 0;
  for (int64_t i = tid & 127; i < a.L; i += 128) {
    if (st.pos[first + i] < 0) continue;
    s += (double)st.loss[first + i], n = 1;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64), n |= __shfl_xor(n, o, 64);
  if ((tid & 63) == 0) sum[tid >> 6] = s, any[tid >> 6] = n;
  __syncthreads();
  const bool counts = (any[0] | any[1] | any[2] | any[3]) != 0;
  float by = 0.f;
  const float loss = counts ? pair_loss(a, (sum[0] + sum[1]) - (sum[2] + sum[3]), pair, by) : 0.f;
  if (tid == 0) {
    each[pair] = loss;
    if (counted != nullptr) counted[pair] = counts ? 1 : 0, bys[pair] = finite_abs(by);
  }
  if (!counts) return;
  for (int64_t i = tid & 127; i < a.L; i += 128) st.z2[first + i] = side == 0 ? by : -by;
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

// The same of a policy's losses, with the largest of the rows' derivatives.
__global__ void __launch_bounds__(1024)
sum_policy_kernel(State st, int T, bool mean, float* out) {
  Close c{0.f, 0.f, 0};
#pragma unroll 4
  for (int i = threadIdx.x; i < T; i += 1024) {
    if (st.pos[i] < 0) continue;
    c.sum += st.loss[i], c.top = fmaxf(c.top, finite_abs(st.z2[i]));
  }
  c = close_up<16>(c);
  if (threadIdx.x != 0) return;
  st.hdr->top = usable(c.top);
  out[0] = mean ? c.sum / (float)max(1, st.hdr->n) : c.sum;
}

// The same of pairs, whose number that count it finds.
__global__ void __launch_bounds__(1024)
sum_pairs_kernel(const float* __restrict__ loss, const int* __restrict__ counted, const float* __restrict__ bys, int64_t pairs,
                 Header* hdr, bool mean, float* out) {
  Close c{0.f, 0.f, 0};
  for (int64_t i = threadIdx.x; i < pairs; i += 1024) c.sum += loss[i], c.top = fmaxf(c.top, bys[i]), c.count += counted[i];
  c = close_up<16>(c);
  if (threadIdx.x != 0) return;
  hdr->count = c.count, hdr->top = usable(c.top);
  out[0] = mean ? c.sum / (float)max(1, c.count) : c.sum;
}

// ------------------------------------------------------------------ gradients
// coef[t] = (c f, 1 - 1 / f) with f = 1 + 2 zl lse, so that a row of dz is
// c f (q - p + p (1 - 1 / f)), and the factors on dw and dh, scale[0] and [1].  One upstream
// gradient for all rows goes into that factor and c = 1: -1 at a label is exact in 16
// bits, where -c would be off by the same rounding in every row.  Otherwise c is the
// row's.  `scaled`: c carries the power of two that brings the largest of them below
// 2^14, and the factors its inverse; or each row's own does, whose inverse is left in
// unscale (0 where dz is 0), and dw's factor undoes that of the copy of the hidden states
// (scale_h_kernel), which brings the largest of those below 2^15.
//
// The loss of a pair is that of `group` rows; weights: null, or each row's derivative by -logp,
// which c carries, but for the largest of them (row_factor).  One workgroup.
__global__ void __launch_bounds__(1024)
coef_kernel(State st, const float* __restrict__ dloss, bool per_row, int group, const float* __restrict__ weights, bool mean,
            float factor, float zl, bool scaled, float2* __restrict__ coef, float* __restrict__ unscale, float* scale) {
  __shared__ float buf[16];
  const int n = st.hdr->n;
  const bool each = scaled && (per_row || weights != nullptr);
  auto c_of = [&](int t) {
    const int row = st.rows[t];
    const float c = per_row ? dloss[group == 1 ? row : row / group] * factor : 1.f;
    return weights != nullptr ? c * weights[row] : c;
  };
  const float top = weights != nullptr && !per_row ? st.hdr->top : 1.f;
  float m = 0.f;
  for (int t = threadIdx.x; t < n; t += 1024) {
    const float c = c_of(t) / top;
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
  const float up = per_row ? 1.f : n == 0 ? 0.f : dloss[0] * factor * (mean ? 1.f / (float)st.hdr->count : 1.f);
  const float f = up * top;
  scale[0] = f / sc, scale[1] = each ? f : f / sc, scale[2] = sc;
}

// The hidden states divided by their rows' powers of two, times dw's (a row a workgroup).
__global__ void __launch_bounds__(256)
scale_h_kernel(State st, const float* __restrict__ unscale, const float* scale, int Dp, f16* __restrict__ out) {
  const int t = blockIdx.x;
  if (t >= st.hdr->n) return;
  const float k = unscale[t] * scale[2];
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

// The workgroup's tile (its number in the order of tile_of's bands) and part: those that are whole
// first, then the parts, one part of all tiles after another; both in contiguous pieces for
// each XCD.  False: it has none.
__device__ __forceinline__ bool dh_work(const DhShare& sh, int tiles, int b, int& id, int& part) {
  const int rest = tiles - sh.whole, all = b < sh.whole ? sh.whole : rest * sh.parts;
  const int i = b < sh.whole ? b : b - sh.whole;
  if (i >= all) return false;
  const int at = xcd_order(i, all);
  id = b < sh.whole ? at : sh.whole + at % rest, part = b < sh.whole ? 0 : at / rest;
  return true;
}

struct DhArgs {
  const char* w;         // at the piece's first row
  const char* dz;
  int64_t ldw, ldz, plane_z;
  int V, Tp, ndt, splits, cols;   // V: rows of w from the piece on; cols: the piece's columns to whole k steps
  float* out;            // [splits][Tp][Dt]
  int Dt;
  bool first;
  bool share;            // tiles are shared by the state's DhShare, `out` is as BwdWs.dh is then
  State st;
};
template <typename C, typename Op, int PZ>
__global__ void __launch_bounds__(C::THREADS, 2)
dh_kernel(DhArgs a) {
  constexpr int BM = C::BM, BN = C::BN;
  using P = Product<Op, BM, BN, C::WM, C::WN, true, false>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS_BYTES];
  const int n = a.st.hdr->n;
  int dt, tt, sp, parts, slot = -1;
  const int row_tiles = (n + BN - 1) / BN;   // of the rows that count, as in logits_kernel
  if (a.share) {
    int id;
    const DhShare sh{a.st.hdr->whole, a.st.hdr->parts};
    if (!dh_work(sh, a.ndt * row_tiles, blockIdx.x, id, sp)) return;
    band_tile(id, a.ndt, row_tiles, dt, tt);
    parts = id < sh.whole ? 1 : sh.parts;
    if (id >= sh.whole) slot = (id - sh.whole) * parts + sp;
  } else {
    const int tiles = gridDim.x / a.splits;
    sp = blockIdx.x / tiles, parts = a.splits;
    const int id = blockIdx.x - sp * tiles;
    if (id >= a.ndt * row_tiles) return;
    tile_of(id, a.ndt, row_tiles, dt, tt);
  }
  const int t0 = tt * BN, d0 = dt * BM;
  const int steps = a.cols / P::BK;
  const int k0 = (int)((int64_t)steps * sp / parts) * P::BK, k1 = (int)((int64_t)steps * (sp + 1) / parts) * P::BK;
  typename P::Acc acc;
  const Operand A{a.w + d0 * P::EB, a.ldw, 0, a.V, (int)a.ldw - d0 * P::EB};
  const Operand B{a.dz + (int64_t)t0 * a.ldz, a.ldz, a.plane_z, a.Tp - t0, a.cols * P::EB};
  P::template run<PZ>(acc, A, B, k0, k1, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / P::WN, wn = wave % P::WN;
  // the tile's corner: in dh itself, in its own copy of it, or in a buffer of the tile's size
  float* corner = slot >= 0 ? a.out + ((int64_t)a.Tp * a.Dt + (int64_t)slot * BM * BN)
                            : a.out + ((int64_t)(a.share ? 0 : sp) * a.Tp + t0) * a.Dt + d0;
  const int ld = slot >= 0 ? BM : a.Dt;
#pragma unroll
  for (int j = 0; j < P::NI; ++j) {
    float* o = corner + (int64_t)(wn * P::NW + 16 * j + (lane & 15)) * ld + wm * P::MW + 4 * (lane >> 4);
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

// dh of every row from what dh_kernel shared out, in the inputs' type (0 for rows that do not count).
// A workgroup per row and 1024 channels, four a thread.
template <typename X>
__global__ void __launch_bounds__(256)
share_out_kernel(State st, const float* __restrict__ dh, int D, int Dt, int Tp, int bn, const float* scale,
                 const float* unscale, X* __restrict__ out) {
  const int64_t row = blockIdx.x;
  const int c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (c >= D) return;
  const int t = st.pos[row];
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (t >= 0) {
    const float f = scale[0] * (unscale != nullptr ? unscale[t] : 1.f);
    const int row_tiles = (st.hdr->n + bn - 1) / bn, tt = t / bn;
    const DhShare sh{st.hdr->whole, st.hdr->parts};
    const int id = band_id(c / kEdge, tt, Dt / kEdge, row_tiles);
    const bool whole = id < sh.whole;
    const float* at = whole ? dh + (int64_t)t * Dt + c
                            : dh + (int64_t)Tp * Dt + (int64_t)(id - sh.whole) * sh.parts * kEdge * bn +
                                  (int64_t)(t - tt * bn) * kEdge + c % kEdge;
    const int parts = whole ? 1 : sh.parts;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(at + (int64_t)i * kEdge * bn);
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
  int V, D, ndt, nvt;    // V: rows of dw from the piece on; nvt: tiles of the piece's columns
  const float* scale;
  void* out;             // dw at the piece's first row
  float* part;           // CUT: [cuts][Vp][Dt]
  int64_t ldp, ldcut;
  int cuts;
  State st;
};
template <typename C, typename Op, typename X, int PZ, bool CUT>
__device__ __forceinline__ void dw_tile(const DwArgs& a, char* lds, int dt, int v0, int cut) {
  constexpr int BM = C::BM, BN = C::BN;
  using P = Product<Op, BM, BN, C::WM, C::WN, true, true>;
  const int n = a.st.hdr->n, d0 = dt * BM;
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

template <typename C, typename Op, typename X, int PZ, bool CUT>
__global__ void __launch_bounds__(C::THREADS, 2)
dw_kernel(DwArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[Product<Op, C::BM, C::BN, C::WM, C::WN, true, true>::LDS_BYTES];
  int dt, vt;
  if constexpr (CUT) {
    const int tiles = gridDim.x / a.cuts, cut = blockIdx.x / tiles;
    tile_of(blockIdx.x - cut * tiles, a.ndt, tiles / a.ndt, dt, vt);
    dw_tile<C, Op, X, PZ, true>(a, lds, dt, vt * C::BN, cut);
  } else if constexpr (__is_same(C, Tile256)) {
    int id, half;
    if (!half_work(a.ndt * a.nvt, blockIdx.x, id, half)) return;
    band_tile(id, a.ndt, a.nvt, dt, vt);
    if (half >= 0) dw_tile<Half256, Op, X, PZ, false>(a, lds, dt, vt * C::BN + half * Half256::BN, 0);
    else dw_tile<C, Op, X, PZ, false>(a, lds, dt, vt * C::BN, 0);
  } else {
    tile_of(blockIdx.x, a.ndt, a.nvt, dt, vt);
    dw_tile<C, Op, X, PZ, false>(a, lds, dt, vt * C::BN, 0);
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
  const int64_t tiles = a.nvt * (up(T, C::BN) / C::BN);
  const int64_t groups = MODE == kCut ? tiles * a.cuts : __is_same(C, Tile256) ? tiles + kHalfMore : tiles;
  logits_kernel<C, Op, MODE, PZ><<<(unsigned)groups, C::THREADS, 0, s>>>(a);
}
// The forward's, whole or in parts.
template <typename C, typename Op>
void launch_forward(const LogitArgs& a, const Plan& p, hipStream_t s) {
  if (p.cuts > 1) launch_logits<C, Op, kCut, 1>(a, p.T, p.Vt, s);
  else launch_logits<C, Op, kStats, 1>(a, p.T, p.Vt, s);
}
template <typename C, typename Op, int PZ>
void launch_dh(DhArgs a, const Plan& p, int room, hipStream_t s) {
  a.ndt = (int)(up(p.D, C::BM) / C::BM);
  const int64_t tiles = a.ndt * (up(p.T, C::BN) / C::BN);
  // (whole tiles and parts: some workgroups have nothing to do, whatever rows count)
  dh_kernel<C, Op, PZ><<<(unsigned)(a.share ? tiles + room : tiles * p.splits), C::THREADS, 0, s>>>(a);
}
template <typename C, typename Op, typename X, int PZ, bool CUT>
void launch_dw(DwArgs a, const Plan& p, int64_t cols, hipStream_t s) {
  a.ndt = (int)(up(p.D, C::BM) / C::BM);
  a.nvt = (int)(cols / C::BN);
  const unsigned tiles = (unsigned)(a.ndt * a.nvt);
  dw_kernel<C, Op, X, PZ, CUT><<<CUT ? tiles * (unsigned)a.cuts : tiles + (__is_same(C, Tile256) ? kHalfMore : 0), C::THREADS, 0,
                                s>>>(a);
  if constexpr (CUT) {
    sum_out_kernel<X, false><<<dim3((unsigned)std::min<int64_t>(cols, a.V), (unsigned)((p.D + 1023) / 1024)), 256, 0, s>>>(
        a.st, a.part, a.D, a.ldp, a.ldcut, a.cuts, a.scale, nullptr, static_cast<X*>(a.out));
  }
}

// What a call computes from the logits.
enum Kind { kLabels, kTeacher, kLogp, kPolicy, kPreference };
struct Loss {
  Kind kind;
  float tau, zl;
  const int64_t* labels;   // null: a teacher, whose entries and rows have been found
  int64_t ignore;
  Policy policy;
  Preference pairs;
};

template <typename X, typename Op>
int forward(const Plan& p, const void* hidden, const void* weight, const State& st, const FwdWs& ws, int K, const Loss& l,
            int reduction, float* loss, hipStream_t s) {
  // the weight too where it is not an operand itself
  const int64_t most = p.copy_w ? std::max(p.T, p.V) : p.T;
  const dim3 packs((unsigned)std::min<int64_t>(8192, most), p.copy_w ? 2 : 1);
  const X* h_in = static_cast<const X*>(hidden);
  const X* w_in = static_cast<const X*>(weight);
  State in = st;
  if (reduction == 0 && l.kind != kPreference) in.loss = loss;   // where rows that do not count leave their 0
  if (l.labels != nullptr && p.T <= kRowsInOne) {
    rows_pack_kernel<X><<<packs, 256, 0, s>>>(h_in, w_in, l.labels, l.ignore, (int)p.T, (int)p.V, (int)p.D, (int)p.Dp, st, in.loss);
  } else {
    if (l.labels != nullptr) rows_kernel<true><<<1, 1024, 0, s>>>(l.labels, l.ignore, p.T, (int)p.V, in);
    else rows_kernel<false><<<1, 1024, 0, s>>>(nullptr, 0, p.T, (int)p.V, in);
    pack_kernel<X><<<packs, 256, 0, s>>>(h_in, w_in, p.V, (int)p.D, (int)p.Dp, st);
  }
  LogitArgs a = logit_args(p, st, weight, K, l.tau);
  a.part = ws.part;
  a.past = keeps_past(p);
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
  const unsigned waves = (unsigned)((p.T + 3) / 4), groups = (unsigned)((p.T + kLogpRows - 1) / kLogpRows);
  float* rows = reduction == 0 ? loss : st.loss;
  const DhShape shape = dh_shape(p);
  if (l.kind == kPreference) {
    row_logp_kernel<false><<<groups, 256, 0, s>>>(st, ws.part, (int)parts, p.Tp, {}, shape, st.loss);
    const int64_t pairs = p.T / (2 * l.pairs.L);
    const bool all = reduction != 0;
    if (p.T <= kTokensInOne) {
      int waves = 16;
      while (waves > 1 && waves * pairs > 16) waves /= 2;
      pairs_kernel<<<1, 1024, 0, s>>>(st, l.pairs, pairs, waves, reduction == 1, all ? nullptr : loss, all ? loss : nullptr);
    } else {
      float* each = all ? reinterpret_cast<float*>(ws.part) : loss;   // two floats a row are there and done with
      int* counted = all ? reinterpret_cast<int*>(each + pairs) : nullptr;
      float* bys = all ? each + 2 * pairs : nullptr;
      pair_kernel<<<(unsigned)pairs, 256, 0, s>>>(st, l.pairs, each, counted, bys);
      if (all) sum_pairs_kernel<<<1, 1024, 0, s>>>(each, counted, bys, pairs, st.hdr, reduction == 1, loss);
    }
    return rr::check_launch("rr_linear_preference");
  }
  if (l.kind == kPolicy) {
    row_logp_kernel<true><<<groups, 256, 0, s>>>(st, ws.part, (int)parts, p.Tp, l.policy, shape, rows);
    if (reduction != 0) sum_policy_kernel<<<1, 1024, 0, s>>>(st, (int)p.T, reduction == 1, loss);
    return rr::check_launch("rr_linear_policy");
  } else if (l.kind == kLogp) {
    row_logp_kernel<false><<<groups, 256, 0, s>>>(st, ws.part, (int)parts, p.Tp, {}, shape, rows);
  } else {
    row_loss_kernel<<<waves, 256, 0, s>>>(st, ws.part, (int)parts, p.Tp, K, l.kind == kLabels, l.zl, l.tau, rows);
  }
  if (reduction != 0) sum_loss_kernel<<<1, 1024, 0, s>>>(st.loss, p.T, st.hdr, reduction == 1, loss);
  return rr::check_launch("rr_linear_loss");
}

// What the backward has to know of a loss: dz is `factor` times (f q - p) and a row's upstream gradient,
// one for `group` rows, and with `weighted` what the forward left for the row.
struct LossGrad {
  float tau, factor, zl;
  int group;
  bool weighted, logp;
};

template <typename X, typename Op, int PZ>
int backward(const Plan& p, const float* dloss, const void* weight, const State& st, const BwdWs& ws, int K, const LossGrad& l,
             int reduction, void* dh, void* dw, hipStream_t s) {
  const bool each = __is_same(Op, OpF16) && (reduction == 0 || l.weighted);   // a power of two for each row's dz
  const bool itself = l.logp && !__is_same(Op, OpF16);   // dz_kernel and logits_kernel find the factors
  const float2* coef = itself ? nullptr : ws.coef;
  const DhShape shape = l.logp ? dh_shape(p) : DhShape{};
  const Upstream us{dloss, l.factor, l.group, reduction == 0, reduction == 1, l.weighted, ws.scale};
  if (!itself) {
    coef_kernel<<<1, 1024, 0, s>>>(st, dloss, reduction == 0, l.group, l.weighted ? st.z2 : nullptr, reduction == 1, l.factor,
                                   l.zl, __is_same(Op, OpF16), ws.coef, ws.unscale, ws.scale);
  }
  if (each && dw != nullptr) {
    scale_h_kernel<<<(unsigned)p.T, 256, 0, s>>>(st, ws.unscale, ws.scale, (int)p.Dp, reinterpret_cast<f16*>(ws.h));
  }
  for (int64_t v = 0; v < p.Vt; v += p.Vp) {
    const int64_t cols = std::min(p.Vp, p.Vt - v);   // whole tiles
    LogitArgs a = logit_args(p, st, weight, K, l.tau);
    a.coef = coef, a.up = us, a.dz = ws.dz, a.ldz = p.Vp * p.eb, a.plane_z = p.Tp * a.ldz, a.v_first = (int)v;
    constexpr bool kFp32 = __is_same(Op, OpF32), kFew = PZ == 2;   // up to kFewRows
    if (kFew || st.z != nullptr) {
      dz_kernel<Op, PZ><<<dim3((unsigned)p.T, (unsigned)(up(cols, kSeg) / kSeg)), 256, 0, s>>>(
          st, coef, us, a.V, p.Vt, K, a.v_first, (int)cols, ws.dz, a.ldz, a.plane_z);
    } else if constexpr (!kFew) {
      launch_logits<typename std::conditional<kFp32, Tile64, Tile256>::type, Op, kGrad, PZ>(a, p.T, cols, s);
    }
    if (dh != nullptr) {
      DhArgs b{};
      b.w = a.w + v * a.ldw, b.dz = ws.dz, b.ldw = a.ldw, b.ldz = a.ldz, b.plane_z = a.plane_z;
      b.V = (int)(p.V - v), b.Tp = a.Tp, b.splits = (int)p.splits, b.cols = (int)cols;
      b.out = ws.dh, b.Dt = (int)p.Dt, b.first = v == 0, b.st = st;
      b.share = l.logp;
      if constexpr (kFew || kFp32) {
        if (p.rows == kTile32) launch_dh<Tile32, Op, PZ>(b, p, shape.room, s);
        else launch_dh<Tile64, Op, PZ>(b, p, shape.room, s);
      } else {
        launch_dh<Tile256, Op, PZ>(b, p, shape.room, s);
      }
    }
    if (dw != nullptr) {
      DwArgs c{};
      c.h = each ? ws.h : st.h, c.dz = ws.dz, c.ldh = a.ldh, c.ldz = a.ldz, c.plane_z = a.plane_z;
      c.V = (int)(p.V - v), c.D = (int)p.D, c.scale = ws.scale;
      c.out = static_cast<X*>(dw) + v * p.D, c.st = st;
      c.part = ws.dw, c.ldp = p.Dt, c.ldcut = p.Vp * p.Dt, c.cuts = (int)p.cuts_w;
      if (kFp32 && l.logp && p.small_w) {
        if constexpr (kFp32) launch_dw<Tile64, Op, X, PZ, false>(c, p, cols, s);
      } else if (kFew || p.cuts_w == 1) {
        launch_dw<Tile256, Op, X, PZ, false>(c, p, cols, s);
      } else if constexpr (!kFew) {
        launch_dw<Tile256, Op, X, PZ, true>(c, p, cols, s);
      }
    }
  }
  if (dh != nullptr && l.logp) {
    share_out_kernel<X><<<dim3((unsigned)p.T, (unsigned)((p.D + 1023) / 1024)), 256, 0, s>>>(
        st, ws.dh, (int)p.D, (int)p.Dt, (int)p.Tp, shape.bn, ws.scale + 1, each ? ws.unscale : nullptr, static_cast<X*>(dh));
  } else if (dh != nullptr) {
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

int run_forward(const void* hidden, const void* weight, int dtype, int64_t T, int64_t D, int64_t V, int64_t K, const Loss& l,
                int reduction, float* loss, const State& st, void* workspace, hipStream_t s) {
  const Plan p = plan_of(T, D, V, dtype);
  FwdWs ws;
  fwd_layout(p, static_cast<char*>(workspace), &ws);
  if (dtype == RR_BF16) return forward<bf16, OpBf16>(p, hidden, weight, st, ws, (int)K, l, reduction, loss, s);
  if (dtype == RR_F16) return forward<f16, OpF16>(p, hidden, weight, st, ws, (int)K, l, reduction, loss, s);
  return forward<float, OpF32>(p, hidden, weight, st, ws, (int)K, l, reduction, loss, s);
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
  return pass == 0 ? fwd_layout(p, nullptr, nullptr) : bwd_layout(p, pass == 2, nullptr, nullptr);
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
  const Loss l{kLabels, 1.f, z_loss, labels, ignore_index};
  return run_forward(hidden, weight, dtype, rows, D, V, 1, l, reduction, loss, st, workspace, s);
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
  const Loss l{kTeacher, temperature, 0.f, nullptr, 0};
  return run_forward(hidden, weight, dtype, rows, D, V, K, l, reduction, loss, st, workspace, s);
}

namespace {

bool bad_temperature(float t) { return !(t > 0.f) || !(t < 1e30f); }

// The forward of the losses on the labels' log-probabilities, `losses` of them where none are added up.
int forward_logp(const char* who, const void* hidden, const void* weight, int dtype, int64_t rows, int64_t D, int64_t V,
                 const Loss& l, int reduction, float* loss, int64_t losses,
                 void* state, size_t state_bytes, void* workspace, size_t workspace_bytes, hipStream_t s) {
  if (int rc = check_dims(who, rows, D, V, 1, dtype, reduction)) return rc;
  const std::string w(who);
  if (bad_temperature(l.tau)) return rr::fail(RR_EINVAL, w + ": temperature must be positive and finite");
  if (losses > 0 || reduction != 0) {
    if (loss == nullptr) return rr::fail(RR_EINVAL, w + ": null pointer");
  }
  if (rows == 0) {
    zero(loss, reduction != 0 ? 4 : losses * 4, s);
    return rr::check_launch(who);
  }
  if (l.labels == nullptr) return rr::fail(RR_EINVAL, w + ": null pointer");
  if (l.kind == kPolicy && (l.policy.advantages == nullptr || (l.policy.kl != 0.f && l.policy.ref == nullptr))) {
    return rr::fail(RR_EINVAL, w + ": null pointer");
  }
  if (int rc = check_buffers(who, rows, D, V, 1, dtype, 0, hidden, weight, state, state_bytes, workspace, workspace_bytes)) return rc;
  State st;
  lay_out_state(rows, D, V, 1, dtype, state, state_bytes, &st);
  return run_forward(hidden, weight, dtype, rows, D, V, 1, l, reduction, loss, st, workspace, s);
}

// The backward of all losses.
int run_backward(const char* who, const float* dloss, const void* weight, int dtype, int64_t rows, int64_t D, int64_t V,
                 int64_t K, const LossGrad& l, int reduction, const void* state, size_t state_bytes, void* dhidden,
                 void* dweight, void* workspace, size_t workspace_bytes, hipStream_t s) {
  if (int rc = check_dims(who, rows, D, V, K, dtype, reduction)) return rc;
  if (bad_temperature(l.tau)) return rr::fail(RR_EINVAL, std::string(who) + ": temperature must be positive and finite");
  const int64_t es = dtype == RR_F32 ? 4 : 2;
  if (rows == 0) {
    zero(dweight, V * D * es, s);
    return rr::check_launch(who);
  }
  if (dloss == nullptr) return rr::fail(RR_EINVAL, std::string(who) + ": null pointer");
  const int pass = l.logp ? 2 : 1;
  if (int rc = check_buffers(who, rows, D, V, K, dtype, pass, nullptr, weight, state, state_bytes, workspace, workspace_bytes)) return rc;
  if (dhidden == nullptr && dweight == nullptr) return RR_OK;
  const Plan p = plan_of(rows, D, V, dtype);
  State st;
  lay_out_state(rows, D, V, K, dtype, const_cast<void*>(state), state_bytes, &st);
  BwdWs ws;
  bwd_layout(p, l.logp, static_cast<char*>(workspace), &ws);
#define LL_BACKWARD(X, OP, PZ) backward<X, OP, PZ>(p, dloss, weight, st, ws, (int)K, l, reduction, dhidden, dweight, s)
  if (dtype == RR_BF16) return p.planes_z == 2 ? LL_BACKWARD(bf16, OpBf16, 2) : LL_BACKWARD(bf16, OpBf16, 1);
  if (dtype == RR_F16) return p.planes_z == 2 ? LL_BACKWARD(f16, OpF16, 2) : LL_BACKWARD(f16, OpF16, 1);
  return LL_BACKWARD(float, OpF32, 1);
#undef LL_BACKWARD
}

}  // namespace

extern "C" int rr_linear_loss_bwd(const float* dloss, const void* weight, int dtype, int64_t rows, int64_t D,
                                  int64_t V, int64_t K, float z_loss, float temperature, int reduction,
                                  const void* state, size_t state_bytes, void* dhidden, void* dweight, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const LossGrad l{temperature, temperature, z_loss, 1, false, false};
  return run_backward("rr_linear_loss_bwd", dloss, weight, dtype, rows, D, V, K, l, reduction, state, state_bytes, dhidden,
                      dweight, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int rr_linear_logp_fwd(const void* hidden, const void* weight, int dtype, int64_t rows, int64_t D, int64_t V,
                                  const int64_t* labels, int64_t ignore_index, float temperature, float* log_probs,
                                  void* state, size_t state_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  const Loss l{kLogp, temperature, 0.f, labels, ignore_index};
  return forward_logp("rr_linear_logp_fwd", hidden, weight, dtype, rows, D, V, l, 0, log_probs, rows,
                      state, state_bytes, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int rr_linear_policy_fwd(const void* hidden, const void* weight, int dtype, int64_t rows, int64_t D, int64_t V,
                                    const int64_t* labels, int64_t ignore_index, float temperature,
                                    const float* advantages, int64_t rows_per_advantage, const float* old_log_probs,
                                    const float* ref_log_probs, float clip_low, float clip_high, float kl_weight,
                                    int reduction, float* loss, void* state, size_t state_bytes, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const std::string w = "rr_linear_policy_fwd";
  if (!(clip_low >= 0.f) || !(clip_high >= 0.f)) return rr::fail(RR_EINVAL, w + ": the clipping's widths must not be negative");
  if (!(kl_weight >= 0.f) || !(kl_weight < INFINITY)) return rr::fail(RR_EINVAL, w + ": kl_weight must be finite and not negative");
  if (rows_per_advantage <= 0) return rr::fail(RR_EINVAL, w + ": an advantage is for one row or more");
  Loss l{kPolicy, temperature, 0.f, labels, ignore_index};
  l.policy = {advantages, rows_per_advantage, old_log_probs, ref_log_probs, 1.f - clip_low, 1.f + clip_high, kl_weight};
  return forward_logp(w.c_str(), hidden, weight, dtype, rows, D, V, l, reduction, loss, rows, state,
                      state_bytes, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int rr_linear_preference_fwd(const void* hidden, const void* weight, int dtype, int64_t pairs, int64_t L,
                                        int64_t D, int64_t V, const int64_t* labels, int64_t ignore_index,
                                        const float* ref_log_probs, float beta, float label_smoothing, int reduction,
                                        float* loss, void* state, size_t state_bytes, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  const std::string w = "rr_linear_preference_fwd";
  if (pairs < 0 || L < 0) return rr::fail(RR_EINVAL, w + ": pairs and tokens must be >= 0");
  if (pairs >= ((int64_t)1 << 23) || L >= ((int64_t)1 << 23)) return rr::fail(RR_EUNSUPPORTED, w + ": too many rows");
  if (!(beta > 0.f) || !(beta < INFINITY)) return rr::fail(RR_EINVAL, w + ": beta must be positive and finite");
  if (!(label_smoothing >= 0.f) || !(label_smoothing <= 0.5f)) return rr::fail(RR_EINVAL, w + ": label_smoothing must be in [0, 0.5]");
  Loss l{kPreference, 1.f, 0.f, labels, ignore_index};
  l.pairs = {ref_log_probs, L, beta, label_smoothing};
  return forward_logp(w.c_str(), hidden, weight, dtype, pairs * 2 * L, D, V, l, reduction, loss, pairs,
                      state, state_bytes, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int rr_linear_logp_bwd(const float* dloss, const void* weight, int dtype, int64_t rows, int64_t D, int64_t V,
                                  float temperature, int64_t rows_per_loss, int of_log_probs, int reduction,
                                  const void* state, size_t state_bytes, void* dhidden, void* dweight, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const std::string w = "rr_linear_logp_bwd";
  if (rows_per_loss <= 0 || rows_per_loss >= ((int64_t)1 << 24)) return rr::fail(RR_EINVAL, w + ": a loss is of one row or more");
  const bool itself = of_log_probs != 0;
  if (itself && (rows_per_loss != 1 || reduction != 0)) {
    return rr::fail(RR_EINVAL, w + ": log-probabilities have a gradient a row");
  }
  // (the log-probabilities' own derivative by -logp is -1)
  const LossGrad l{temperature, (itself ? -1.f : 1.f) / temperature, 0.f, (int)rows_per_loss, !itself, true};
  return run_backward(w.c_str(), dloss, weight, dtype, rows, D, V, 1, l, reduction, state, state_bytes, dhidden, dweight,
                      workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}
