// Global gradient norm over many tensors, and clipping by it.
//
//   total = sqrt(sum over all tensors and elements of g^2)
//   g     = g * min(1, max_norm / (total + eps))
//
// One launch covers up to PER tensors: their addresses and sizes travel in the kernel's arguments
// (nothing is copied to the device, and a captured graph holds them by value).  The squares are
// summed in 64 bits: an fp32 square leaves its range for |g| above 1.8e19 or below 1e-22, and the
// sum runs over up to 1e10 elements.  Partial sums are written per workgroup and joined in a fixed
// order, by every workgroup of the clip for itself (16 KB of them for up to 1024 tensors, 2 KB more for each
// further 128; a launch of its own for that would cost a small list a third of its time): no atomics, the same
// bits every time.
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.h"

namespace {
constexpr int NT = 256;
constexpr int PER = 128;            // tensors per launch (kernel arguments stay under 4 KiB)
constexpr int CHUNK = 16384;        // elements a workgroup takes at a time
constexpr int NORM_GRID = 2048, NORM_LEAST = 256, CLIP_GRID = 2048;

struct Tensors {
  const void* src[PER];
  void* dst[PER];
  int64_t n[PER];                   // elements | type << 60
  int first[PER + 1];               // chunks before tensor i
  int count;
};

__device__ __forceinline__ int owner(const Tensors& t, int chunk) {
  int lo = 0, hi = t.count;         // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// 16-byte vectors with the element's alignment: a gradient that is a view into a flat buffer may
// start anywhere
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(N)));
  typedef type at __attribute__((aligned(sizeof(T))));
};

template <typename T>
__device__ __forceinline__ double sum_squares(const T* p, int len) {
  constexpr int N = Vec<T>::N, STEP = NT * N;
  double s = 0.0;
  int i = threadIdx.x * N;
  for (; i + 3 * STEP + N <= len; i += 4 * STEP) {
    typename Vec<T>::type v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = *(const typename Vec<T>::at*)(p + i + u * STEP);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const double d = (double)(float)v[u][k];
        s = fma(d, d, s);
      }
  }
  for (; i < len; i += STEP)
    for (int k = 0; k < N && i + k < len; ++k) {
      const double d = (double)(float)p[i + k];
      s = fma(d, d, s);
    }
  return s;
}

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += red[i];
  return s;
}
__device__ __forceinline__ double sum_parts(const double* __restrict__ part, int P, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < P; i += NT) s += part[i];
  return block_sum_f64(s, red);
}

__global__ __launch_bounds__(NT) void grads_norm_kernel(Tensors t, double* __restrict__ part) {
  __shared__ double red[NT / 64];
  double s = 0.0;
  for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int i = owner(t, c);
    const int64_t n = t.n[i] & ((1ll << 60) - 1), at = (int64_t)(c - t.first[i]) * CHUNK;
    const int len = (int)(n - at < CHUNK ? n - at : CHUNK), type = (int)(t.n[i] >> 60);
    if (type == 0) s += sum_squares((const float*)t.src[i] + at, len);
    else if (type == 1) s += sum_squares((const bf16*)t.src[i] + at, len);
    else s += sum_squares((const _Float16*)t.src[i] + at, len);
  }
  s = block_sum_f64(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ __launch_bounds__(NT) void grads_norm_join_kernel(const double* __restrict__ part, int P,
                                                             double* __restrict__ sumsq) {
  __shared__ double red[NT / 64];
  const double s = sum_parts(part, P, red);
  if (threadIdx.x == 0) sumsq[0] = s;
}

// The factor as f * post, post a power of two.  It is formed in fp32 where that holds it (post 1); a norm past
// the largest fp32 (gradients of 1e38) or a factor below its smallest normal number goes through 64 bits and keeps its
// digits in f, since what it scales need not be small: 1e38 clipped to a norm of 1 is an ordinary number.
struct Factor {
  float f, post;
};
__device__ __forceinline__ Factor factor(double total, float max_norm, float eps) {
  const float c = max_norm / ((float)total + eps);
  if (c >= 0x1p-126f || !(total < __builtin_huge_val())) return {c > 1.f ? 1.f : c, 1.f};   // a NaN norm stays NaN
  const double d = max_norm / (total + eps);
  if (!(d < 1.0)) return {1.f, 1.f};               // and 0 / 0, whose gradients are all zeros
  if (d >= 0x1p-126) return {(float)d, 1.f};
  return {(float)(d * 0x1p126), 0x1p-126f};
}

// Vectors of 16 bytes of the wider type, so that a store instruction writes whole lines (bf16 to fp32
// over 0.8 G elements: 1.18 ms with the norm, against 1.24 with 16-byte loads and two stores each),
// four loads in flight per thread (one: 1.30 ms, eight: 1.19).
template <typename TS, typename TD>
__device__ __forceinline__ void scaled(const TS* src, TD* dst, int len, Factor by) {
  constexpr int N = 16 / (sizeof(TS) > sizeof(TD) ? sizeof(TS) : sizeof(TD)), AHEAD = 4, STEP = NT * N;
  typedef TS svec __attribute__((ext_vector_type(N)));
  typedef svec sat __attribute__((aligned(sizeof(TS))));
  typedef TD dvec __attribute__((ext_vector_type(N)));
  typedef dvec dat __attribute__((aligned(sizeof(TD))));
  int i = threadIdx.x * N;
  for (; i + (AHEAD - 1) * STEP + N <= len; i += AHEAD * STEP) {
    svec v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) v[u] = *(const sat*)(src + i + u * STEP);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      dvec o;
#pragma unroll
      for (int k = 0; k < N; ++k) o[k] = (TD)((float)v[u][k] * by.f * by.post);
      *(dat*)(dst + i + u * STEP) = o;
    }
  }
  for (; i < len; i += STEP)
    for (int k = i; k < len && k < i + N; ++k) dst[k] = (TD)((float)src[k] * by.f * by.post);
}

// dst = src * factor; norm_out gets the norm once (infinity past fp32).  In place with a factor of 1 nothing
// changes, so nothing is read.
__global__ __launch_bounds__(NT) void grads_clip_kernel(Tensors t, int dtype,
                                                        const double* __restrict__ part, int P,
                                                        float max_norm, float eps,
                                                        float* __restrict__ norm_out) {
  __shared__ double red[NT / 64];
  const double total = sqrt(sum_parts(part, P, red));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)total;
  const Factor by = factor(total, max_norm, eps);
  if (dtype < 0 && by.f == 1.f && by.post == 1.f) return;
  for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int i = owner(t, c);
    const int64_t n = t.n[i] & ((1ll << 60) - 1), at = (int64_t)(c - t.first[i]) * CHUNK;
    const int len = (int)(n - at < CHUNK ? n - at : CHUNK), type = (int)(t.n[i] >> 60);
    const int to = dtype < 0 ? type : dtype;
    auto run = [&](auto* src) {
      if (to == 0) scaled(src + at, (float*)t.dst[i] + at, len, by);
      else if (to == 1) scaled(src + at, (bf16*)t.dst[i] + at, len, by);
      else scaled(src + at, (_Float16*)t.dst[i] + at, len, by);
    };
    if (type == 0) run((const float*)t.src[i]);
    else if (type == 1) run((const bf16*)t.src[i]);
    else run((const _Float16*)t.src[i]);
  }
}

// calls f(Tensors) for each launch's share of the list; false if an entry cannot be served
template <typename F>
bool for_each_launch(const void* const* src, void* const* dst, const int64_t* n, const int32_t* type,
                     int64_t count, F f) {
  Tensors t;
  t.count = 0;
  t.first[0] = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (n[i] < 0 || type[i] < 0 || type[i] > 2 || (n[i] > 0 && (!src[i] || (dst && !dst[i])))) return false;
    if (n[i] == 0) continue;
    const int64_t chunks = (n[i] + CHUNK - 1) / CHUNK;
    if (chunks > (1 << 30)) return false;
    if (t.count == PER || t.first[t.count] + chunks > (1 << 30)) {
      f(t);
      t.count = 0;
    }
    t.src[t.count] = src[i];
    t.dst[t.count] = dst ? dst[i] : nullptr;
    t.n[t.count] = n[i] | ((int64_t)type[i] << 60);
    t.first[t.count + 1] = t.first[t.count] + (int)chunks;
    ++t.count;
  }
  if (t.count) f(t);
  return true;
}
int grid_of(const Tensors& t, int most) {
  const int c = t.first[t.count];
  return c < most ? c : most;
}
// workgroups per launch of the norm, so that all launches' partial sums stay few
int norm_grid(int64_t live) {
  const int64_t g = NORM_GRID / ((live + PER - 1) / PER);
  return (int)(g < NORM_LEAST ? NORM_LEAST : g);
}
// the partial sums of the list's launches; how many
int norm_parts(const void* const* grads, const int64_t* n, const int32_t* type, int64_t count, double* part,
               hipStream_t s) {
  int64_t live = 0;
  for (int64_t i = 0; i < count; ++i) live += n[i] > 0;
  int P = 0;
  if (live)
    for_each_launch(grads, nullptr, n, type, count, [&](const Tensors& t) {
      const int g = grid_of(t, norm_grid(live));
      hipLaunchKernelGGL(grads_norm_kernel, dim3(g), dim3(NT), 0, s, t, part + P);
      P += g;
    });
  return P;
}
bool bad_list(const void* const* src, void* const* dst, const int64_t* n, const int32_t* type, int64_t count) {
  return count < 0 || (count && (!src || !n || !type)) ||
         !for_each_launch(src, dst, n, type, count, [](const Tensors&) {});
}
}  // namespace

extern "C" int64_t prfl_grads_parts(const int64_t* n, int64_t count) {
  int64_t chunks = 0, live = 0;
  for (int64_t i = 0; i < count; ++i)
    if (n[i] > 0) chunks += (n[i] + CHUNK - 1) / CHUNK, ++live;
  if (!live) return 0;
  // a launch ends after PER tensors or 2^30 chunks
  const int64_t most = ((live + PER - 1) / PER + chunks / (1 << 29)) * norm_grid(live);
  return chunks < most ? chunks : most;
}

extern "C" int prfl_grads_overlap(const void* const* grads, const int64_t* n, const int32_t* type, int64_t count) {
  if (count <= 0 || !grads || !n || !type) return 0;
  try {
    std::vector<uintptr_t> start, end;
    for (int64_t i = 0; i < count; ++i)
      if (n[i] > 0) {
        start.push_back((uintptr_t)grads[i]);
        end.push_back(start.back() + (uintptr_t)n[i] * (type[i] ? 2 : 4));
      }
    std::sort(start.begin(), start.end());
    std::sort(end.begin(), end.end());
    // apart if and only if the i-th end is not past the start after the i-th
    for (size_t i = 0; i + 1 < start.size(); ++i)
      if (end[i] > start[i + 1]) return 1;
  } catch (...) {
    return 1;                       // no memory for the lists
  }
  return 0;
}

extern "C" int prfl_grads_sumsq(const void* const* grads, const int64_t* n, const int32_t* type,
                                int64_t count, double* part, int64_t parts, double* sumsq,
                                void* stream) {
  if (!sumsq || bad_list(grads, nullptr, n, type, count) || parts < prfl_grads_parts(n, count) ||
      (parts && !part))
    return (int)hipErrorInvalidValue;
  hipStream_t s = (hipStream_t)stream;
  const int P = norm_parts(grads, n, type, count, part, s);
  hipLaunchKernelGGL(grads_norm_join_kernel, dim3(1), dim3(NT), 0, s, part, P, sumsq);
  PRFL_LAUNCH_CHECK();
  return 0;
}

extern "C" int prfl_grads_clip(const void* const* grads, void* const* out, const int64_t* n,
                               const int32_t* type, int64_t count, int out_type, const double* sumsq,
                               double* part, int64_t parts, float max_norm, float eps, float* norm,
                               void* stream) {
  void* const* dst = out ? out : (void* const*)grads;
  if (out_type > 2 || (out_type >= 0) != (out != nullptr) || bad_list(grads, dst, n, type, count) ||
      !(max_norm >= 0.f) || !(eps >= 0.f) || (!sumsq && (parts < prfl_grads_parts(n, count) || (parts && !part))))
    return (int)hipErrorInvalidValue;
  hipStream_t s = (hipStream_t)stream;
  const int P = sumsq ? 1 : norm_parts(grads, n, type, count, part, s);
  const double* total = sumsq ? sumsq : part;
  bool first = true;
  auto launch = [&](const Tensors& t) {
    const int g = grid_of(t, CLIP_GRID);
    hipLaunchKernelGGL(grads_clip_kernel, dim3(g < 1 ? 1 : g), dim3(NT), 0, s, t, out_type, total, P,
                       max_norm, eps, first ? norm : nullptr);
    first = false;
  };
  for_each_launch(grads, dst, n, type, count, launch);
  if (first && norm) {              // nothing but empty tensors: the norm alone
    Tensors none;
    none.count = 0;
    none.first[0] = 0;
    launch(none);
  }
  PRFL_LAUNCH_CHECK();
  return 0;
}
