// grad_norm.hip — the norm of many tensors taken together, and their scaling down to a
// largest norm, on gfx950.
//
//   n = sqrt(sum over all tensors of g^2);  f = max / n where n > max, else 1;  out = f g
//
// Two launches for up to 128 tensors: the first leaves a partial sum a workgroup, every
// workgroup of the second adds those up (in the same order, so all have the same f) and
// scales its share.  The table of tensors travels in the kernels' arguments: nothing is copied
// to the device and nothing waits, so a call can be captured in a graph.  Neighbours in
// memory are one entry of it: 301 pieces of one flat buffer are two launches, not six.
//
// What bounds it: HBM.  The gradients are read twice, since no value can be scaled before all are
// summed.  The second reading finds in the 256 MB cache what the first left there last: the
// second goes from the end to the start, what comes earlier than the last 256 MB is read past the
// cache, and so is all of the output written (483 M values of bf16, 965 MB: 552 us with
// ordinary loads and stores, 524 with the stores past the cache, 480 as it is, 6.0 TB/s of all
// three passes; the norm alone 170 and 147 us, 6.6 TB/s).
//
// Sums are in 64 bits, and so is the product: squares of any fp32 value neither overflow nor
// vanish, and what is left is the rounding to the output's type (16 bits: through fp32, which adds up
// to 2^-24 of the value).
#include "rr_common.h"

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

namespace {

using rr::bf16;
using rr::f16;

constexpr int kTensors = 128;      // of a launch: the table is below the 4 KiB that arguments may take
constexpr int kThreads = 256;
constexpr int kVec = 8;            // values a thread takes at a time
constexpr int kStep = kThreads * kVec;
// Workgroups of all launches together, four a CU (16, 30, 60 and 250 M values of bf16: 22, 32, 60 and 240
// us; with eight 24, 35, 61 and 239).
constexpr int kGroups = 1024;
constexpr int64_t kCacheBytes = 256 << 20;
// From so many bytes on the second reading's loads go past the cache, whose lines they are the last to
// want (bf16, 16, 30, 60, 100 and 250 M values: 22, 34, 60, 96 and 240 us past it, 21, 32, 60, 98 and 245 not).
constexpr int64_t kLastBytes = 128 << 20;
constexpr int kDeep = 2;           // loads on their way at one time (4: 488 us where 2 take 480)

struct Table {
  const void* in[kTensors];
  void* out[kTensors];
  int64_t n[kTensors];
  int first[kTensors + 1];         // chunks of the tensors in front of each
  uint8_t type[kTensors];
  int tensors, chunk;              // values of a chunk
  int warm;                        // first chunk that the cache is to keep for the second reading
};
static_assert(sizeof(Table) <= 3800, "arguments of a launch");

// The tensor of a chunk: the last whose first chunk is not behind it.
__device__ __forceinline__ int tensor_of(const Table& t, int c) {
  int lo = 0, hi = t.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Eight values as they lie in memory, from any element on.
template <typename X>
struct Eight {
  typedef uint32_t Words __attribute__((ext_vector_type(2 * sizeof(X))));
  typedef Words Any __attribute__((aligned(sizeof(X))));
  X v[kVec];
  template <bool PAST>   // the cache
  __device__ __forceinline__ void load(const X* p) {
    const Any* at = reinterpret_cast<const Any*>(p);
    const Words w = PAST ? __builtin_nontemporal_load(at) : *at;
    __builtin_memcpy(v, &w, sizeof(w));
  }
  __device__ __forceinline__ void store(X* p) const {
    Words w;
    __builtin_memcpy(&w, v, sizeof(w));
    __builtin_nontemporal_store(w, reinterpret_cast<Any*>(p));
  }
};

__device__ __forceinline__ double wave_add(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Of the whole workgroup, to all of its threads.
__device__ __forceinline__ double group_add(double v, double* buf) {
  v = wave_add(v);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  return (buf[0] + buf[1]) + (buf[2] + buf[3]);
}

template <bool PAST, typename X>
__device__ __forceinline__ double squares(const X* p, int n) {
  double a[4] = {0, 0, 0, 0};
  int i = threadIdx.x * kVec;
  for (; i + (kDeep - 1) * kStep + kVec <= n; i += kDeep * kStep) {
    Eight<X> x[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) x[d].template load<PAST>(p + i + d * kStep);
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const double g = (double)rr::to_f32(x[d].v[e]);
        a[e & 3] = fma(g, g, a[e & 3]);
      }
  }
  for (; i + kVec <= n; i += kStep) {
    Eight<X> x;
    x.template load<PAST>(p + i);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const double g = (double)rr::to_f32(x.v[e]);
      a[e & 3] = fma(g, g, a[e & 3]);
    }
  }
  for (int e = 0; i + e < n && e < kVec; ++e) {
    const double g = (double)rr::to_f32(p[i + e]);
    a[0] = fma(g, g, a[0]);
  }
  return (a[0] + a[1]) + (a[2] + a[3]);
}

template <typename X>
__device__ __forceinline__ X scaled(X g, double f) { return rr::from_f32<X>((float)((double)rr::to_f32(g) * f)); }

template <bool PAST, typename X>
__device__ __forceinline__ void scale(const X* p, X* o, int n, double f) {
  int i = threadIdx.x * kVec;
  for (; i + (kDeep - 1) * kStep + kVec <= n; i += kDeep * kStep) {
    Eight<X> x[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) x[d].template load<PAST>(p + i + d * kStep);
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[d].v[e] = scaled(x[d].v[e], f);
      x[d].store(o + i + d * kStep);
    }
  }
  for (; i + kVec <= n; i += kStep) {
    Eight<X> x;
    x.template load<PAST>(p + i);
#pragma unroll
    for (int e = 0; e < kVec; ++e) x.v[e] = scaled(x.v[e], f);
    x.store(o + i);
  }
  for (int e = 0; i + e < n && e < kVec; ++e) o[i + e] = scaled(p[i + e], f);
}

// What a chunk is: its tensor, where it starts there and how many values it has.
struct Chunk {
  int i, n;
  int64_t at;
};
__device__ __forceinline__ Chunk chunk_of(const Table& t, int c) {
  Chunk k;
  k.i = __builtin_amdgcn_readfirstlane(tensor_of(t, c));
  k.at = (int64_t)(c - t.first[k.i]) * t.chunk;
  k.n = (int)min((int64_t)t.chunk, t.n[k.i] - k.at);
  return k;
}

template <bool PAST>
__device__ __forceinline__ double chunk_squares(const Table& t, const Chunk& k) {
  const void* p = t.in[k.i];
  if (t.type[k.i] == RR_F32) return squares<PAST>(static_cast<const float*>(p) + k.at, k.n);
  if (t.type[k.i] == RR_BF16) return squares<PAST>(static_cast<const bf16*>(p) + k.at, k.n);
  return squares<PAST>(static_cast<const f16*>(p) + k.at, k.n);
}

__global__ void __launch_bounds__(kThreads)
squares_kernel(Table t, int chunks, double* __restrict__ part) {
  __shared__ double buf[4];
  double s = 0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const Chunk k = chunk_of(t, c);
    s += c < t.warm ? chunk_squares<true>(t, k) : chunk_squares<false>(t, k);
  }
  s = group_add(s, buf);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm from the partial sums, by a workgroup.
__device__ __forceinline__ double norm_of(const double* __restrict__ part, int parts, double* buf) {
  double s = 0;
  for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
  return sqrt(group_add(s, buf));
}

__global__ void __launch_bounds__(kThreads)
norm_kernel(const double* __restrict__ part, int parts, float* norm) {
  __shared__ double buf[4];
  const double n = norm_of(part, parts, buf);
  if (threadIdx.x == 0) *norm = (float)n;
}

// The last chunks come first: they are what the cache still holds of the first launch.
template <bool PAST>
__global__ void __launch_bounds__(kThreads)
scale_kernel(Table t, int chunks, const double* __restrict__ part, int parts, double most, float* norm) {
  __shared__ double buf[4];
  const double n = norm_of(part, parts, buf);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const double f = n > most && n < INFINITY ? most / n : 1.;
  for (int c = chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const Chunk k = chunk_of(t, c);
    const void* p = t.in[k.i];
    void* o = t.out[k.i];
    if (f == 1. && p == o) continue;
    if (t.type[k.i] == RR_F32) scale<PAST>(static_cast<const float*>(p) + k.at, static_cast<float*>(o) + k.at, k.n, f);
    else if (t.type[k.i] == RR_BF16) scale<PAST>(static_cast<const bf16*>(p) + k.at, static_cast<bf16*>(o) + k.at, k.n, f);
    else scale<PAST>(static_cast<const f16*>(p) + k.at, static_cast<f16*>(o) + k.at, k.n, f);
  }
}

// ------------------------------------------------------------------ host
struct Launch {
  Table table;
  int chunks, groups;
};

int64_t bytes_of(int64_t n, int dtype) { return n * (dtype == RR_F32 ? 4 : 2); }

int check_tensors(const char* who, int64_t count, const void* const* grads, const int64_t* numel, const int* dtypes) {
  const std::string w(who);
  if (count < 0 || count > (1 << 24)) return rr::fail(RR_EINVAL, w + ": 0 to 2^24 tensors");
  if (count > 0 && (grads == nullptr || numel == nullptr || dtypes == nullptr)) return rr::fail(RR_EINVAL, w + ": null pointer");
  for (int64_t i = 0; i < count; ++i) {
    if (!rr::valid_dtype(dtypes[i])) return rr::fail(RR_EINVAL, w + ": unsupported dtype");
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 48)) return rr::fail(RR_EINVAL, w + ": a tensor's size is out of range");
    if (numel[i] == 0) continue;
    if (grads[i] == nullptr) return rr::fail(RR_EINVAL, w + ": null pointer");
    if (reinterpret_cast<uintptr_t>(grads[i]) % bytes_of(1, dtypes[i]) != 0) return rr::fail(RR_EINVAL, w + ": misaligned tensor");
  }
  return RR_OK;
}

// Tensors one behind the other in memory, in and out: one run of values.
struct Run {
  const char* in;
  char* out;
  int64_t n;
  int type;
  int64_t bytes() const { return bytes_of(n, type); }
};
int runs_of(const char* who, int64_t count, const void* const* grads, void* const* out, const int64_t* numel,
            const int* dtypes, std::vector<Run>* runs) {
  const std::string w(who);
  for (int64_t i = 0; i < count; ++i) {
    if (numel[i] == 0) continue;
    const char* in = static_cast<const char*>(grads[i]);
    char* to = out == nullptr ? nullptr : static_cast<char*>(out[i]);
    if (out != nullptr) {
      if (to == nullptr) return rr::fail(RR_EINVAL, w + ": null pointer");
      if (reinterpret_cast<uintptr_t>(to) % bytes_of(1, dtypes[i]) != 0) return rr::fail(RR_EINVAL, w + ": misaligned tensor");
    }
    if (!runs->empty()) {
      Run& r = runs->back();
      if (r.type == dtypes[i] && in == r.in + r.bytes() && (out == nullptr || to == r.out + r.bytes())) {
        r.n += numel[i];
        continue;
      }
    }
    runs->push_back({in, to, numel[i], dtypes[i]});
  }
  return RR_OK;
}

// What is written must not be another's: neither written nor read.
int check_disjoint(const char* who, const std::vector<Run>& runs) {
  const std::string w(who);
  struct Range {
    uintptr_t at, end;
  };
  std::vector<Range> written;
  written.reserve(runs.size());
  for (const Run& r : runs) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(r.out);
    written.push_back({at, at + (uintptr_t)r.bytes()});
  }
  auto before = [](const Range& a, const Range& b) { return a.at < b.at; };
  if (!std::is_sorted(written.begin(), written.end(), before)) std::sort(written.begin(), written.end(), before);
  for (size_t k = 1; k < written.size(); ++k)
    if (written[k].at < written[k - 1].end) return rr::fail(RR_EINVAL, w + ": two of the tensors to write share memory");
  for (const Run& r : runs) {
    if (r.in == r.out) continue;   // (what is written in place shares nothing, as just seen)
    const uintptr_t at = reinterpret_cast<uintptr_t>(r.in), end = at + (uintptr_t)r.bytes();
    auto k = std::upper_bound(written.begin(), written.end(), at, [](uintptr_t v, const Range& x) { return v < x.end; });
    if (k != written.end() && k->at < end) return rr::fail(RR_EINVAL, w + ": a tensor to write shares memory with another to read");
  }
  return RR_OK;
}

int64_t launches_of(int64_t count) { return std::max<int64_t>(1, (count + kTensors - 1) / kTensors); }

// The launches over the tensors.  Chunks are of 2048 to 16384 values, so that many small tensors make
// enough of them and large ones not too many to look up (of 4096 at most: 567 us where it takes 478); workgroups
// are in proportion to chunks.  *bytes: of all values.
int plan(const char* who, const std::vector<Run>& runs, std::vector<Launch>* launches, int64_t* bytes) {
  int64_t total = 0;
  *bytes = 0;
  for (const Run& r : runs) total += r.n, *bytes += r.bytes();
  int chunk = kStep;
  while (chunk < 8 * kStep && total / chunk > 4 * kGroups) chunk *= 2;
  int64_t chunks = 0;
  for (const Run& r : runs) chunks += (r.n + chunk - 1) / chunk;
  if (chunks >= ((int64_t)1 << 31)) return rr::fail(RR_EUNSUPPORTED, std::string(who) + ": too many values");
  Launch l{};
  auto flush = [&] {
    const Table& t = l.table;
    if (t.tensors == 0) return;
    l.chunks = t.first[t.tensors];
    l.groups = (int)std::min<int64_t>(l.chunks, std::max<int64_t>(1, kGroups * (int64_t)l.chunks / chunks));
    launches->push_back(l);
    l = Launch{};
  };
  int64_t cold = *bytes - kCacheBytes;   // what is left of the bytes that the cache is not to keep
  for (const Run& r : runs) {
    Table& t = l.table;
    const int mine = (int)((r.n + chunk - 1) / chunk);
    t.chunk = chunk;
    t.in[t.tensors] = r.in, t.out[t.tensors] = r.out, t.n[t.tensors] = r.n, t.type[t.tensors] = (uint8_t)r.type;
    t.first[t.tensors + 1] = t.first[t.tensors] + mine;
    if (cold > 0) t.warm = t.first[t.tensors] + (int)std::min<int64_t>(mine, cold / bytes_of(chunk, r.type));
    cold -= r.bytes();
    if (++t.tensors == kTensors) flush();
  }
  flush();
  return RR_OK;
}

int run_norm(const std::vector<Launch>& launches, double* part, hipStream_t s) {
  int parts = 0;
  for (const Launch& l : launches) {
    squares_kernel<<<(unsigned)l.groups, kThreads, 0, s>>>(l.table, l.chunks, part + parts);
    parts += l.groups;
  }
  return parts;
}

int check_workspace(const char* who, int64_t count, const void* ws, size_t ws_bytes, const float* norm) {
  const std::string w(who);
  if (norm == nullptr || ws == nullptr) return rr::fail(RR_EINVAL, w + ": null pointer");
  if (ws_bytes < rr_grad_norm_workspace_bytes(count)) return rr::fail(RR_EWORKSPACE, w + ": workspace too small");
  if (reinterpret_cast<uintptr_t>(ws) % 16 != 0) return rr::fail(RR_EWORKSPACE, w + ": workspace misaligned");
  return RR_OK;
}

// (std::vector may throw; nothing leaves a C entry)
template <typename F>
int guarded(const char* who, F f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return rr::fail(RR_EINVAL, std::string(who) + ": " + e.what());
  }
}

}  // namespace

extern "C" size_t rr_grad_norm_workspace_bytes(int64_t count) {
  if (count < 0 || count > (1 << 24)) return 0;
  return (size_t)(kGroups + launches_of(count)) * sizeof(double);   // a launch's share of the workgroups is at least one
}

extern "C" int rr_grad_norm(int64_t count, const void* const* grads, const int64_t* numel, const int* dtypes, float* norm,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "rr_grad_norm";
  return guarded(who, [&]() -> int {
    if (int rc = check_tensors(who, count, grads, numel, dtypes)) return rc;
    if (int rc = check_workspace(who, count, workspace, workspace_bytes, norm)) return rc;
    std::vector<Run> runs;
    std::vector<Launch> launches;
    int64_t bytes = 0;
    if (int rc = runs_of(who, count, grads, nullptr, numel, dtypes, &runs)) return rc;
    if (int rc = plan(who, runs, &launches, &bytes)) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    double* part = static_cast<double*>(workspace);
    const int parts = run_norm(launches, part, s);
    norm_kernel<<<1, kThreads, 0, s>>>(part, parts, norm);
    return rr::check_launch(who);
  });
}

extern "C" int rr_clip_grad_norm(int64_t count, const void* const* grads, void* const* out, const int64_t* numel,
                                 const int* dtypes, double max_norm, float* norm, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  const char* who = "rr_clip_grad_norm";
  return guarded(who, [&]() -> int {
    if (int rc = check_tensors(who, count, grads, numel, dtypes)) return rc;
    if (!(max_norm >= 0)) return rr::fail(RR_EINVAL, std::string(who) + ": max_norm must not be negative");
    if (count > 0 && out == nullptr) return rr::fail(RR_EINVAL, std::string(who) + ": null pointer");
    if (int rc = check_workspace(who, count, workspace, workspace_bytes, norm)) return rc;
    std::vector<Run> runs;
    std::vector<Launch> launches;
    int64_t bytes = 0;
    if (int rc = runs_of(who, count, grads, out, numel, dtypes, &runs)) return rc;
    if (int rc = check_disjoint(who, runs)) return rc;
    if (int rc = plan(who, runs, &launches, &bytes)) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    double* part = static_cast<double*>(workspace);
    const int parts = run_norm(launches, part, s);
    if (launches.empty()) norm_kernel<<<1, kThreads, 0, s>>>(part, 0, norm);
    for (size_t k = launches.size(); k-- > 0;) {
      const Launch& l = launches[k];
      float* n = k == 0 ? norm : nullptr;
      if (bytes >= kLastBytes) scale_kernel<true><<<(unsigned)l.groups, kThreads, 0, s>>>(l.table, l.chunks, part, parts, max_norm, n);
      else scale_kernel<false><<<(unsigned)l.groups, kThreads, 0, s>>>(l.table, l.chunks, part, parts, max_norm, n);
    }
    return rr::check_launch(who);
  });
}
