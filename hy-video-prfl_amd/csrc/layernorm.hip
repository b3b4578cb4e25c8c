// Layer norm over the last axis, forward and backward, for any width up to 16384, any row stride
// and fp32 / bf16 / fp16 in and out.
//
//   mu = sum_c x / C,  v = sum_c (x - mu)^2 / C,  r = 1 / sqrt(v + eps),  xhat = (x - mu) r
//   y  = xhat w + b                                       (w, b each optional)
//   g  = dy w,   dx = r (g - sum_c g / C - xhat sum_c (g xhat) / C)
//   dw = sum over rows of dy xhat,   db = sum over rows of dy
//
// A row is read once and held in registers: the statistics, the output and the gradients come
// from there.  All statistics and sums are fp32; y and dx are rounded once, to their own type;
// dw and db stay fp32.
#include <math.h>

#include "common.h"

namespace {
constexpr int MAXC = 16384;
constexpr int MAXT = 1024;    // threads per row at most
constexpr int MAXW = MAXT / 64;

template <typename T>
struct Chunk {                 // 16 bytes of a row
  static constexpr int N = 16 / sizeof(T);
};

// N values from p, the first n of them real (the others 0).  Rows of odd width or stride are not
// aligned to 16 bytes: the vector is declared with the element's alignment, which gfx950 loads
// and stores whole.
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, int n, float (&v)[N]) {
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec uvec __attribute__((aligned(sizeof(T))));
  if (n >= N) {
    const vec t = *(const uvec*)p;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, int n, const float (&v)[N]) {
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec uvec __attribute__((aligned(sizeof(T))));
  if (n >= N) {
    vec t;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = (T)v[i];
    *(uvec*)p = t;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}
template <int N>
__device__ __forceinline__ void load_any(const void* p, int type, int64_t at, int n, float (&v)[N]) {
  if (type == 0) load_n<float, N>((const float*)p + at, n, v);
  else if (type == 1) load_n<bf16, N>((const bf16*)p + at, n, v);
  else load_n<_Float16, N>((const _Float16*)p + at, n, v);
}

// mean and rstd of a row held as v[NV][N] per thread.  Within a wave two passes over the
// registers; across waves the partial sums of squares about the waves' own means are joined:
//   M2 = sum_w M2_w + n_w (mu_w - mu)^2,
// so a mean far from zero costs no digits.  red: the row's [waves][2] floats, double-buffered by
// the caller so that one barrier a row is enough.
template <int NV, int N>
__device__ __forceinline__ void row_stats(const float (&v)[NV][N], const int (&cnt)[NV], int C, int nw,
                                          int wave_n, float eps, float* red, float& mean,
                                          float& rstd) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) s += v[j][i];
  s = wave_sum(s);
  const float mw = wave_n > 0 ? s / wave_n : 0.f;
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = i < cnt[j] ? v[j][i] - mw : 0.f;
      q += d * d;
    }
  q = wave_sum(q);
  if (nw == 1) {
    mean = mw;
  } else {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      red[3 * w] = s;
      red[3 * w + 1] = q;
      red[3 * w + 2] = (float)wave_n;
    }
    __syncthreads();
    s = 0.f;
    for (int i = 0; i < nw; ++i) s += red[3 * i];
    mean = s / C;
    q = 0.f;
    for (int i = 0; i < nw; ++i) {
      const float n = red[3 * i + 2];
      const float d = n > 0.f ? red[3 * i] / n - mean : 0.f;
      q += red[3 * i + 1] + n * d * d;
    }
  }
  rstd = 1.f / sqrtf(q / C + eps);
}

// One row per workgroup at a time (nw waves), or per wave (nw == 1, four rows per workgroup).
template <typename TX, typename TY, int NV>
__global__ __launch_bounds__(MAXT) void layer_norm_fwd_kernel(
    const TX* __restrict__ x, int64_t ldx, int64_t rows, int C, const void* __restrict__ w,
    const void* __restrict__ b, int wtype, float eps, TY* __restrict__ y, int64_t ldy,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int nw) {
  constexpr int N = Chunk<TX>::N;
  __shared__ float red[2][3 * MAXW];
  const int T = nw * 64, per = nw == 1 ? blockDim.x / 64 : 1;
  const int t = nw == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int first = t & ~63;                       // the wave's first chunk in each stripe
  int cnt[NV], wave_n = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    cnt[j] = min(max(C - (t + j * T) * N, 0), N);
    wave_n += min(max(C - (first + j * T) * N, 0), 64 * N);
  }
  float wv[NV][N], bv[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < N; ++i) wv[j][i] = 1.f, bv[j][i] = 0.f;
    if (w) load_any<N>(w, wtype, (int64_t)(t + j * T) * N, cnt[j], wv[j]);
    if (b) load_any<N>(b, wtype, (int64_t)(t + j * T) * N, cnt[j], bv[j]);
  }
  int64_t row = (int64_t)blockIdx.x * per + (nw == 1 ? threadIdx.x >> 6 : 0);
  for (int it = 0; row < rows; row += (int64_t)gridDim.x * per, ++it) {
    float v[NV][N], mean, rstd;
#pragma unroll
    for (int j = 0; j < NV; ++j) load_n<TX, N>(x + row * ldx + (t + j * T) * N, cnt[j], v[j]);
    row_stats<NV, N>(v, cnt, C, nw, wave_n, eps, red[it & 1], mean, rstd);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float o[N];
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fmaf((v[j][i] - mean) * rstd, wv[j][i], bv[j][i]);
      store_n<TY, N>(y + row * ldy + (t + j * T) * N, cnt[j], o);
    }
    if (t == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

// dx of each row and, where asked for, the workgroup's sums of dy xhat and dy over its rows
// (part_w / part_b [gridDim.x][C]).
template <typename TX, typename TY, int NV, int TMAX>
__global__ __launch_bounds__(TMAX) void layer_norm_bwd_kernel(
    const TY* __restrict__ dy, int64_t lddy, const TX* __restrict__ x, int64_t ldx,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, int64_t rows, int C,
    const void* __restrict__ w, int wtype, TX* __restrict__ dx, int64_t lddx,
    float* __restrict__ part_w, float* __restrict__ part_b, int nw) {
  constexpr int N = Chunk<TX>::N;
  __shared__ float red[2][2 * MAXW];
  __shared__ float join[4][64 * N];
  const int T = nw * 64, per = nw == 1 ? blockDim.x / 64 : 1;
  const int t = nw == 1 ? threadIdx.x & 63 : threadIdx.x, wv_id = threadIdx.x >> 6;
  int cnt[NV];
  float wv[NV][N], sw[NV][N], sb[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    cnt[j] = min(max(C - (t + j * T) * N, 0), N);
#pragma unroll
    for (int i = 0; i < N; ++i) wv[j][i] = 1.f, sw[j][i] = 0.f, sb[j][i] = 0.f;
    if (w) load_any<N>(w, wtype, (int64_t)(t + j * T) * N, cnt[j], wv[j]);
  }
  int64_t row = (int64_t)blockIdx.x * per + (nw == 1 ? wv_id : 0);
  for (int it = 0; row < rows; row += (int64_t)gridDim.x * per, ++it) {
    const float mean = mean_in[row], rstd = rstd_in[row];
    float xh[NV][N], g[NV][N], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      load_n<TX, N>(x + row * ldx + (t + j * T) * N, cnt[j], xh[j]);
      load_n<TY, N>(dy + row * lddy + (t + j * T) * N, cnt[j], g[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        xh[j][i] = (xh[j][i] - mean) * rstd;
        sw[j][i] = fmaf(g[j][i], xh[j][i], sw[j][i]);
        sb[j][i] += g[j][i];
        g[j][i] *= wv[j][i];
        s1 += g[j][i];
        s2 = fmaf(g[j][i], xh[j][i], s2);
      }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if (nw > 1) {
      float* r = red[it & 1];
      if ((threadIdx.x & 63) == 0) r[2 * wv_id] = s1, r[2 * wv_id + 1] = s2;
      __syncthreads();
      s1 = s2 = 0.f;
      for (int i = 0; i < nw; ++i) s1 += r[2 * i], s2 += r[2 * i + 1];
    }
    const float m1 = s1 / C, m2 = s2 / C;
    if (dx) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float o[N];
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = rstd * (g[j][i] - m1 - xh[j][i] * m2);
        store_n<TX, N>(dx + row * lddx + (t + j * T) * N, cnt[j], o);
      }
    }
  }
  // the four waves of a wave-per-row workgroup hold the same columns: wave 0 adds them in order
  auto put = [&](float* part, float (&s)[NV][N]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (nw == 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) join[wv_id][i * 64 + t] = s[j][i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i)
          s[j][i] = join[0][i * 64 + t] + join[1][i * 64 + t] + join[2][i * 64 + t] + join[3][i * 64 + t];
      }
      if (nw > 1 || wv_id == 0)
        store_n<float, N>(part + (int64_t)blockIdx.x * C + (t + j * T) * N, cnt[j], s[j]);
    }
  };
  if (part_w) put(part_w, sw);
  if (part_b) put(part_b, sb);
}

// out[c] = sum over p of part[p][c] for up to two [P][C] matrices (blockIdx.y): 64 columns per
// workgroup, its 16 waves taking every 16th row, joined in a fixed order.
__global__ __launch_bounds__(1024) void layer_norm_dw_kernel(const float* __restrict__ part0,
                                                             const float* __restrict__ part1, int P,
                                                             int C, float* __restrict__ out0,
                                                             float* __restrict__ out1) {
  __shared__ float red[16][64];
  const float* part = blockIdx.y ? part1 : part0;
  float* out = blockIdx.y ? out1 : out0;
  if (!part) return;
  const int l = threadIdx.x & 63, wv = threadIdx.x >> 6, c = blockIdx.x * 64 + l;
  float s = 0.f;
  if (c < C)
    for (int p = wv; p < P; p += 16) s += part[(int64_t)p * C + c];
  red[wv][l] = s;
  __syncthreads();
  if (wv == 0 && c < C) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += red[i][l];
    out[c] = s;
  }
}

// waves and chunks per thread for a row of C elements, at most 16 elements a thread
struct Split {
  int nv, nw;
};
Split split_for(int C, int x_type) {
  const int n = x_type ? 8 : 4, most = 16 / n, chunks = (C + n - 1) / n;
  int nv = 1;
  while (nv < most && chunks > 256 * nv) ++nv;
  return {nv, (chunks + 64 * nv - 1) / (64 * nv)};
}
int grid_for_rows(int64_t rows, int nw, int64_t most) {
  const int64_t per = nw == 1 ? 4 : 1, g = (rows + per - 1) / per;
  return (int)(g < most ? g : most);
}

template <typename F>
int by_types(int xt, int yt, F f) {
  const float* a = nullptr;
  const bf16* b = nullptr;
  const _Float16* h = nullptr;
  switch (xt * 3 + yt) {
    case 0: return f(a, a);
    case 1: return f(a, b);
    case 2: return f(a, h);
    case 3: return f(b, a);
    case 4: return f(b, b);
    case 5: return f(b, h);
    case 6: return f(h, a);
    case 7: return f(h, b);
    default: return f(h, h);
  }
}
template <int MOST, typename F>
void by_nv(int nv, F f) {
  if (nv == 1) f(std::integral_constant<int, 1>());
  else if (nv == 2) f(std::integral_constant<int, 2>());
  else if constexpr (MOST > 2) {
    if (nv == 3) f(std::integral_constant<int, 3>());
    else f(std::integral_constant<int, 4>());
  }
}
bool bad(int64_t rows, int64_t C, int xt, int yt, int wt) {
  return rows < 0 || C < 1 || C > MAXC || xt < 0 || xt > 2 || yt < 0 || yt > 2 || wt < 0 || wt > 2;
}
constexpr int64_t BWD_PARTS = 512;
}  // namespace

extern "C" int64_t prfl_layer_norm_parts(int64_t rows, int64_t C, int x_type) {
  if (bad(rows, C, x_type, 0, 0)) return 0;
  const Split s = split_for((int)C, x_type);
  return grid_for_rows(rows, s.nw, BWD_PARTS);
}

extern "C" int prfl_layer_norm_fwd(const void* x, int x_type, int64_t ldx, int64_t rows, int64_t C,
                                   const void* w, const void* b, int w_type, float eps, void* y,
                                   int y_type, int64_t ldy, float* mean, float* rstd, void* stream) {
  if (bad(rows, C, x_type, y_type, w_type) || (rows > 1 && (ldx < 0 || ldy < C)) || !(eps >= 0.f))
    return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  if (!x || !y || !mean || !rstd) return (int)hipErrorInvalidValue;
  hipStream_t s = (hipStream_t)stream;
  const Split sp = split_for((int)C, x_type);
  prfl_prof::begin(KID_LN, s);
  by_types(x_type, y_type, [&](auto* tx, auto* ty) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(tx)>>;
    using TY = std::remove_const_t<std::remove_pointer_t<decltype(ty)>>;
    by_nv<16 / Chunk<TX>::N>(sp.nv, [&](auto nv) {
      hipLaunchKernelGGL((layer_norm_fwd_kernel<TX, TY, nv()>), dim3(grid_for_rows(rows, sp.nw, 2048)),
                         dim3(sp.nw == 1 ? 256 : sp.nw * 64), 0, s, (const TX*)x, ldx, rows, (int)C, w,
                         b, w_type, eps, (TY*)y, ldy, mean, rstd, sp.nw);
    });
    return 0;
  });
  prfl_prof::set_work((double)rows * C * ((x_type ? 2 : 4) + (y_type ? 2 : 4)));
  prfl_prof::end(KID_LN, s);
  PRFL_LAUNCH_CHECK();
  return 0;
}

extern "C" int prfl_layer_norm_bwd(const void* dy, int y_type, int64_t lddy, const void* x, int x_type,
                                   int64_t ldx, const float* mean, const float* rstd, int64_t rows,
                                   int64_t C, const void* w, int w_type, void* dx, int64_t lddx,
                                   float* dw, float* db, float* part, void* stream) {
  if (bad(rows, C, x_type, y_type, w_type) || (rows > 1 && (ldx < 0 || lddy < 0 || (dx && lddx < C))) ||
      ((dw || db) && !part))
    return (int)hipErrorInvalidValue;
  hipStream_t s = (hipStream_t)stream;
  const Split sp = split_for((int)C, x_type);
  const int grid = rows ? grid_for_rows(rows, sp.nw, BWD_PARTS) : 0;
  float* pw = dw ? part : nullptr;
  float* pb = db ? part + (dw ? (int64_t)grid * C : 0) : nullptr;
  prfl_prof::begin(KID_LN, s);
  if (rows && (dx || dw || db)) {
    if (!dy || !x || !mean || !rstd) return (int)hipErrorInvalidValue;
    by_types(x_type, y_type, [&](auto* tx, auto* ty) {
      using TX = std::remove_const_t<std::remove_pointer_t<decltype(tx)>>;
      using TY = std::remove_const_t<std::remove_pointer_t<decltype(ty)>>;
      by_nv<16 / Chunk<TX>::N>(sp.nv, [&](auto nv) {
        auto kernel = layer_norm_bwd_kernel<TX, TY, nv(), 512>;
        if constexpr (nv() * Chunk<TX>::N == 16)      // rows past 8192 elements: more than 8 waves
          if (sp.nw > 8) kernel = layer_norm_bwd_kernel<TX, TY, nv(), MAXT>;
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(sp.nw == 1 ? 256 : sp.nw * 64), 0, s,
                           (const TY*)dy, lddy, (const TX*)x, ldx, mean, rstd, rows, (int)C, w, w_type,
                           (TX*)dx, lddx, pw, pb, sp.nw);
      });
      return 0;
    });
  }
  if (dw || db)
    hipLaunchKernelGGL(layer_norm_dw_kernel, dim3((C + 63) / 64, 2), dim3(1024), 0, s, pw, pb, grid,
                       (int)C, dw, db);
  prfl_prof::set_work((double)rows * C * (2 * (x_type ? 2 : 4) + (y_type ? 2 : 4)));
  prfl_prof::end(KID_LN, s);
  PRFL_LAUNCH_CHECK();
  return 0;
}
