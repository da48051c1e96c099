// layer_norm.hip — layer norm over the last axis on gfx950, forward and backward.
//
//   forward   mu = mean(x);  r = 1 / sqrt(mean((x - mu)^2) + eps);  xh = (x - mu) r
//             y = xh w + b
//   backward  g = dy w;  dx = r (g - mean(g) - xh mean(g xh))
//             dw = sum over rows of dy xh;  db = sum over rows of dy
//
// The rows are streamed once: a row stays in the registers of its threads (up to 8192
// channels, below) between the statistics and the output, so the variance is that of the
// differences (two passes over registers, no cancellation) and HBM sees x (and
// dy) once and y (dx) once.  The kernels are bound by those bytes, a single
// token by its launch.
//
// A row belongs to TPR threads, eight consecutive elements per thread and step: a wave,
// whose sums need no barrier, while its registers hold the row, else a workgroup.
// Reached on an MI355X (a 2 GiB copy: 4.9 TB/s): 32768 x 2560 bf16 forward 4.8 TB/s,
// backward 4.6 TB/s, the reduction of the parameters' gradients included; 1536 x 768
// 5 and 11 us, one token 5 us, launches mostly.  A workgroup a row: backward 5.0 TB/s at
// 16384 x 5120, 3.3 at 16384 x 2688 (a third of the lanes idle); beyond 8192 channels its 1024
// threads' registers spill: 2.7 TB/s at 4096 x 16384, 0.7 at 2048 x 32768.
// Rows start at any element (odd D): the 16-byte accesses are made at the
// element type's alignment, which global memory allows, and only a row's last
// piece is element by element.
//
// The weight's and bias's gradients: each thread of the backward owns fixed
// columns and adds them up over its rows in fp32, a workgroup leaves one partial
// row, and ln_param_kernel adds the partial rows in a fixed order (no atomics:
// the same inputs give the same bits).
#include "rr_common.h"
#include "rr_mfma.h"

#include <algorithm>
#include <string>

namespace {

using rr::bf16;
using rr::f16;

constexpr int64_t kMaxChannels = 32768;   // 1024 threads, 4 steps of 8 elements
constexpr int kPartRows = 512;            // partial rows of dw and db at most
// Workgroups of a forward launch at most: HIP launches fewer than 2^32 threads.  (One launch whose
// workgroups stride over the rows took 97 us in place of 68 at 32768 x 2560: the loop
// keeps the weight and the bias in registers.)
constexpr int64_t kMaxBlocks = 1 << 21;

// Eight consecutive elements as they lie in memory (any alignment of T).
template <typename T>
struct Raw {
  typedef uint32_t Words __attribute__((ext_vector_type(2 * sizeof(T))));
  Words w;
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
    else return rr::to_f32(__builtin_bit_cast(T, (uint16_t)(w[e / 2] >> (16 * (e % 2)))));
  }
  // Columns c .. c + 7 of a row of D (0 past its end).
  __device__ __forceinline__ void load(const T* row, int c, int D) {
    if (c + 8 <= D) {
      typedef Words Any __attribute__((aligned(sizeof(T))));
      w = *reinterpret_cast<const Any*>(row + c);
      return;
    }
#pragma unroll
    for (int i = 0; i < (int)(2 * sizeof(T)); ++i) w[i] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (c + e >= D) continue;
      if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(row[c + e]);
      else w[e / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, row[c + e]) << (16 * (e % 2));
    }
  }
};
template <typename T>
__device__ __forceinline__ void load_cols(const T* row, int c, int D, float (&v)[8]) {
  Raw<T> r;
  r.load(row, c, D);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = r.get(e);
}
template <typename T>
__device__ __forceinline__ void store_cols(T* row, int c, int D, const float (&v)[8]) {
  if (c + 8 <= D) {
    typedef typename Raw<T>::Words Words;
    typedef Words Any __attribute__((aligned(sizeof(T))));
    Words w;
#pragma unroll
    for (int i = 0; i < (int)(2 * sizeof(T)); ++i) {
      if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
      else if constexpr (__is_same(T, bf16)) w[i] = rr::bf_pack2(v[2 * i], v[2 * i + 1]);
      else w[i] = __builtin_bit_cast(uint16_t, rr::from_f32<T>(v[2 * i])) |
                  (uint32_t)__builtin_bit_cast(uint16_t, rr::from_f32<T>(v[2 * i + 1])) << 16;
    }
    *reinterpret_cast<Any*>(row + c) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < D) row[c + e] = rr::from_f32<T>(v[e]);
  }
}
// The weight or bias, of any of the three types (one uniform branch a piece), or `fill` where there is none.
__device__ __forceinline__ void load_param(const void* p, int dtype, int c, int D, float fill, float (&v)[8]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fill;
  } else if (dtype == RR_F32) {
    load_cols(static_cast<const float*>(p), c, D, v);
  } else if (dtype == RR_BF16) {
    load_cols(static_cast<const bf16*>(p), c, D, v);
  } else {
    load_cols(static_cast<const f16*>(p), c, D, v);
  }
}

// Sums of a and b over the TPR threads of a row, in every thread (the same bits
// in each).  TPR > 64: a workgroup, through `buf` (2 floats a wave).
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* buf) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o, 64), b += __shfl_xor(b, o, 64);
  if constexpr (TPR > 64) {
    const int w = threadIdx.x >> 6;
    __syncthreads();   // the last sum's reads of buf are done
    if ((threadIdx.x & 63) == 0) buf[2 * w] = a, buf[2 * w + 1] = b;
    __syncthreads();
    a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) a += buf[2 * i], b += buf[2 * i + 1];
  }
}

template <int TPR> constexpr int block_threads() { return TPR == 64 ? 256 : TPR; }

// One row per TPR threads; NV pieces of 8 elements per thread.
template <typename X, typename Y, int TPR, int NV>
__global__ void __launch_bounds__(block_threads<TPR>())
ln_fwd_kernel(const X* __restrict__ x, const void* w, const void* b, int wdt, int64_t rows, int D, float eps,
              Y* __restrict__ y, float* mean, float* rstd) {
  __shared__ float buf[2 * (TPR / 64)];
  constexpr int RPB = block_threads<TPR>() / TPR;
  const int lane = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= rows) return;   // a whole wave (TPR 64), or no row at all
  const X* xr = x + row * D;
  float v[NV][8];
  float s = 0.f, zero = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) load_cols(xr, (j * TPR + lane) * 8, D, v[j]);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[j][e];
  row_sum2<TPR>(s, zero, buf);
  const float inv = 1.f / (float)D;
  const float mu = s * inv;
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = (j * TPR + lane) * 8 + e < D ? v[j][e] - mu : 0.f;
      v[j][e] = d;
      q += d * d;
    }
  zero = 0.f;
  row_sum2<TPR>(q, zero, buf);
  const float r = 1.f / sqrtf(q * inv + eps);
  if (mean != nullptr && lane == 0) mean[row] = mu, rstd[row] = r;
  Y* yr = y + row * D;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * 8;
    if (c >= D) break;
    float wv[8], bv[8], o[8];
    load_param(w, wdt, c, D, 1.f, wv);
    load_param(b, wdt, c, D, 0.f, bv);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = v[j][e] * r * wv[e] + bv[e];
    store_cols(yr, c, D, o);
  }
}

// Rows strided over the grid, the next row's loads issued ahead of this row's sums; dw
// and db partials of the workgroup's rows in part[block][2][D] (null: not wanted).
template <typename X, typename Y, int TPR, int NV>
__global__ void __launch_bounds__(block_threads<TPR>())
ln_bwd_kernel(const Y* __restrict__ dy, const X* __restrict__ x, const void* w, int wdt, const float* mean,
              const float* rstd, int64_t rows, int D, X* __restrict__ dx, float* __restrict__ part) {
  __shared__ float buf[2 * (TPR / 64)];
  constexpr int RPB = block_threads<TPR>() / TPR;
  __shared__ float cols[RPB > 1 ? (RPB - 1) * 64 * 8 : 1];
  const int lane = threadIdx.x % TPR;
  const int slot = threadIdx.x / TPR;
  float wv[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + lane) * 8;
    if (c < D) load_param(w, wdt, c, D, 1.f, wv[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (c >= D) wv[j][e] = 0.f;
      dw[j][e] = 0.f, db[j][e] = 0.f;
    }
  }
  const float inv = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + slot;
  Raw<X> xn[NV];
  Raw<Y> gn[NV];
  float mn = 0.f, rn = 0.f;
  auto fetch = [&](int64_t r) {
    mn = mean[r], rn = rstd[r];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      xn[j].load(x + r * D, (j * TPR + lane) * 8, D);
      gn[j].load(dy + r * D, (j * TPR + lane) * 8, D);
    }
  };
  if (row < rows) fetch(row);
  for (; row < rows; row += step) {
    Raw<X> xc[NV];
    Raw<Y> gc[NV];
    const float mu = mn, r = rn;
#pragma unroll
    for (int j = 0; j < NV; ++j) xc[j] = xn[j], gc[j] = gn[j];
    if (row + step < rows) fetch(row + step);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = gc[j].get(e);     // 0 past the row's end
        const float h = (xc[j].get(e) - mu) * r;
        const float g = d * wv[j][e];
        db[j][e] += d, s1 += g;
        dw[j][e] += d * h, s2 += g * h;
      }
    if (dx != nullptr) {
      row_sum2<TPR>(s1, s2, buf);
      s1 *= inv, s2 *= inv;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + lane) * 8;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = r * (gc[j].get(e) * wv[j][e] - s1 - (xc[j].get(e) - mu) * r * s2);
        if (c < D) store_cols(dx + row * D, c, D, o);
      }
    }
  }
  if (part == nullptr) return;
  float* pw = part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float(&acc)[8] = h == 0 ? dw[j] : db[j];
      if constexpr (RPB > 1) {   // the waves of the workgroup, in order
        __syncthreads();
        if (slot > 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) cols[((slot - 1) * 8 + e) * 64 + lane] = acc[e];
        }
        __syncthreads();
        if (slot == 0) {
          for (int q = 0; q < RPB - 1; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += cols[(q * 8 + e) * 64 + lane];
        }
      }
      const int c = (j * TPR + lane) * 8;
      if (slot == 0 && c < D) store_cols(pw + h * D, c, D, acc);
    }
}

// dw and db from the partial rows: a workgroup takes 64 columns of one of them, its
// sixteen waves every sixteenth partial row, added up in order.
__global__ void __launch_bounds__(1024)
ln_param_kernel(const float* __restrict__ part, int n, int D, void* dw, void* db, int wdt) {
  __shared__ float buf[16][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int c = blockIdx.x * 64 + lane, h = blockIdx.y;
  void* out = h == 0 ? dw : db;
  if (out == nullptr) return;
  float s = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int i = wave; i < n; i += 16) s += part[((int64_t)i * 2 + h) * D + c];
  }
  buf[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= D) return;
  for (int i = 1; i < 16; ++i) s += buf[i][lane];
  if (wdt == RR_F32) static_cast<float*>(out)[c] = s;
  else if (wdt == RR_BF16) static_cast<bf16*>(out)[c] = rr::from_f32<bf16>(s);
  else static_cast<f16*>(out)[c] = rr::from_f32<f16>(s);
}

// Threads a row and pieces a thread for D channels.  A wave a row (no barrier) while its
// registers hold the row: 8 pieces forward, 5 backward (3 of fp32), where the next row and
// the parameters' sums are held too.  32768 x 2560 bf16: 74 and 111 us; with a workgroup a
// row 87 and 146 us.
constexpr int wave_pieces(bool bwd, bool fp32) { return !bwd ? 8 : fp32 ? 3 : 5; }
struct Shape { int tpr, nv; };
Shape shape_of(int64_t D, bool bwd, bool fp32) {
  const int64_t v = (D + 7) / 8;   // pieces of a row
  const int tpr = v <= 64 * wave_pieces(bwd, fp32) ? 64 : v <= 256 * 4 ? 256 : 1024;
  return {tpr, (int)((v + tpr - 1) / tpr)};
}
// Whether shape_of gives this one.
constexpr bool reached(bool bwd, bool fp32, int tpr, int nv) {
  const int w = wave_pieces(bwd, fp32);
  return tpr == 64 ? nv <= w : tpr == 256 ? nv <= 4 && nv * 256 > w * 64 : nv <= 4 && nv * 1024 > 1024;
}
// Workgroups of the backward: two rows a wave (or workgroup) where that leaves fewer than
// kPartRows partial rows.
int64_t bwd_blocks(int64_t rows, int64_t D, bool fp32) {
  const int64_t rpb = shape_of(D, true, fp32).tpr == 64 ? 8 : 2;
  return std::max<int64_t>(1, std::min<int64_t>(kPartRows, (rows + rpb - 1) / rpb));
}

int check_args(const char* who, int64_t rows, int64_t D, int xdt, int ydt, int wdt) {
  const std::string w(who);
  if (rows < 0 || D <= 0) return rr::fail(RR_EINVAL, w + ": rows must be >= 0 and D > 0");
  if (D > kMaxChannels) return rr::fail(RR_EUNSUPPORTED, w + ": at most " + std::to_string(kMaxChannels) +
                                                             " channels, got " + std::to_string(D));
  if (!rr::valid_dtype(xdt) || !rr::valid_dtype(ydt) || !rr::valid_dtype(wdt)) {
    return rr::fail(RR_EINVAL, w + ": unsupported dtype");
  }
  if (ydt != xdt && xdt != RR_F32) return rr::fail(RR_EINVAL, w + ": y has x's dtype, or any where x is fp32");
  if (rows >= ((int64_t)1 << 31)) return rr::fail(RR_EUNSUPPORTED, w + ": too many rows");
  return RR_OK;
}

}  // namespace

#define LN_CASE(BWD, TPR, NV, KERNEL, NB, ...)                                                                   \
  case NV:                                                                                                       \
    if constexpr (reached(BWD, sizeof(X) == 4, TPR, NV)) KERNEL<X, Y, TPR, NV><<<NB, block_threads<TPR>(), 0, s>>>(__VA_ARGS__); \
    break;
#define LN_NV(BWD, TPR, ...)                                                                                     \
  switch (sh.nv) {                                                                                               \
    LN_CASE(BWD, TPR, 1, __VA_ARGS__) LN_CASE(BWD, TPR, 2, __VA_ARGS__) LN_CASE(BWD, TPR, 3, __VA_ARGS__)        \
    LN_CASE(BWD, TPR, 4, __VA_ARGS__) LN_CASE(BWD, TPR, 5, __VA_ARGS__) LN_CASE(BWD, TPR, 6, __VA_ARGS__)        \
    LN_CASE(BWD, TPR, 7, __VA_ARGS__) LN_CASE(BWD, TPR, 8, __VA_ARGS__)                                          \
  }
#define LN_SHAPE(BWD, ...)                                                                                       \
  if (sh.tpr == 64) { LN_NV(BWD, 64, __VA_ARGS__) }                                                              \
  else if (sh.tpr == 256) { LN_NV(BWD, 256, __VA_ARGS__) }                                                       \
  else { LN_NV(BWD, 1024, __VA_ARGS__) }
// x and y types: the same, or fp32 x with any y.
#define LN_TYPES(...)                                                                                            \
  if (x_dtype == RR_BF16) { using X = bf16; using Y = bf16; __VA_ARGS__ }                                        \
  else if (x_dtype == RR_F16) { using X = f16; using Y = f16; __VA_ARGS__ }                                      \
  else if (y_dtype == RR_F32) { using X = float; using Y = float; __VA_ARGS__ }                                  \
  else if (y_dtype == RR_BF16) { using X = float; using Y = bf16; __VA_ARGS__ }                                  \
  else { using X = float; using Y = f16; __VA_ARGS__ }

extern "C" int rr_layer_norm_fwd(const void* x, int x_dtype, const void* w, const void* b, int w_dtype, int64_t rows,
                                 int64_t D, float eps, void* y, int y_dtype, float* mean, float* rstd, void* stream) {
  if (int rc = check_args("rr_layer_norm_fwd", rows, D, x_dtype, y_dtype, w_dtype)) return rc;
  if (!(eps >= 0.f)) return rr::fail(RR_EINVAL, "rr_layer_norm_fwd: eps must not be negative");
  if (rows == 0) return RR_OK;
  if (x == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr)) {
    return rr::fail(RR_EINVAL, "rr_layer_norm_fwd: null pointer");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Shape sh = shape_of(D, false, x_dtype == RR_F32);
  const int64_t rpb = sh.tpr == 64 ? 4 : 1;
  for (int64_t r = 0; r < rows; r += kMaxBlocks * rpb) {
    const int64_t n = std::min(rows - r, kMaxBlocks * rpb);
    float* const mean_r = mean == nullptr ? nullptr : mean + r;
    float* const rstd_r = mean == nullptr ? nullptr : rstd + r;
    const int nb = (int)((n + rpb - 1) / rpb);
    LN_TYPES(LN_SHAPE(false, ln_fwd_kernel, nb, static_cast<const X*>(x) + r * D, w, b, w_dtype, n, (int)D, eps,
                      static_cast<Y*>(y) + r * D, mean_r, rstd_r))
  }
  return rr::check_launch("rr_layer_norm_fwd");
}

extern "C" size_t rr_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t D) {
  if (rows <= 0 || D <= 0 || D > kMaxChannels) return 0;
  return (size_t)bwd_blocks(rows, D, true) * 2 * (size_t)D * sizeof(float);   // fp32's, at least those of 16 bits
}

extern "C" int rr_layer_norm_bwd(const void* dy, int y_dtype, const void* x, int x_dtype, const void* w, int w_dtype,
                                 const float* mean, const float* rstd, int64_t rows, int64_t D, void* dx, void* dw,
                                 void* db, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_args("rr_layer_norm_bwd", rows, D, x_dtype, y_dtype, w_dtype)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool params = dw != nullptr || db != nullptr;
  const int64_t nb = rows == 0 ? 0 : bwd_blocks(rows, D, x_dtype == RR_F32);
  if (rows > 0) {
    if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr) {
      return rr::fail(RR_EINVAL, "rr_layer_norm_bwd: null pointer");
    }
    if (params && (workspace == nullptr || workspace_bytes < rr_layer_norm_bwd_workspace_bytes(rows, D))) {
      return rr::fail(RR_EWORKSPACE, "rr_layer_norm_bwd: workspace too small");
    }
    if (params && reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
      return rr::fail(RR_EWORKSPACE, "rr_layer_norm_bwd: workspace misaligned");
    }
    if (!params && dx == nullptr) return RR_OK;
    float* part = params ? static_cast<float*>(workspace) : nullptr;
    const Shape sh = shape_of(D, true, x_dtype == RR_F32);
    LN_TYPES(LN_SHAPE(true, ln_bwd_kernel, (int)nb, static_cast<const Y*>(dy), static_cast<const X*>(x), w, w_dtype, mean, rstd,
                      rows, (int)D, static_cast<X*>(dx), part))
  }
  if (params) {
    const dim3 grid((unsigned)((D + 63) / 64), 2);
    ln_param_kernel<<<grid, 1024, 0, s>>>(static_cast<const float*>(workspace), (int)nb, (int)D, dw, db, w_dtype);
  }
  return rr::check_launch("rr_layer_norm_bwd");
}
