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
constexpr int NARROW = 256;   // threads of a workgroup whose rows take a wave or less each

// N values of a row as they lie in memory.  Rows of odd width or stride are not aligned to 16 bytes: the
// vector is declared with the element's alignment, which gfx950 loads and stores whole.
template <typename T, int N>
struct Raw {
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec at __attribute__((aligned(sizeof(T))));
};
template <typename T>
constexpr int CHUNK = 16 / sizeof(T);          // 16 bytes of x

// N values from p, the first n of them real (the others 0)
template <typename T, int N>
__device__ __forceinline__ typename Raw<T, N>::vec load_raw(const T* p, int n) {
  typename Raw<T, N>::vec t;
  if (n >= N) {
    t = *(const typename Raw<T, N>::at*)p;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = i < n ? p[i] : (T)0.f;
  }
  return t;
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, int n, const float (&v)[N]) {
  if (n >= N) {
    typename Raw<T, N>::vec t;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = (T)v[i];
    *(typename Raw<T, N>::at*)p = t;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}
template <int N>
__device__ __forceinline__ void load_any(const void* p, int type, int64_t at, int n, float (&v)[N]) {
  auto widen = [&](auto raw) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)raw[i];
  };
  if (type == 0) widen(load_raw<float, N>((const float*)p + at, n));
  else if (type == 1) widen(load_raw<bf16, N>((const bf16*)p + at, n));
  else widen(load_raw<_Float16, N>((const _Float16*)p + at, n));
}

// mean and rstd of a row held as v[NV][N] per thread.  Within a wave two passes over the
// registers; across waves the partial sums of squares about the waves' own means are joined:
//   M2 = sum_w M2_w + n_w (mu_w - mu)^2,
// so a mean far from zero costs no digits.  red: the row's [waves][2] floats, double-buffered by
// the caller so that one barrier a row is enough.
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int NV, int N, int LANES>
__device__ __forceinline__ void row_stats(const float (&v)[NV][N], const int (&cnt)[NV], int C, int nw,
                                          int wave_n, float eps, float* red, float& mean,
                                          float& rstd) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) s += v[j][i];
  s = row_sum<LANES>(s);
  const float mw = wave_n > 0 ? s / wave_n : 0.f;
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = i < cnt[j] ? v[j][i] - mw : 0.f;
      q += d * d;
    }
  q = row_sum<LANES>(q);
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

// One row per workgroup at a time (nw waves), or with nw == 1 per LANES lanes (64, or 32 / 16 for rows
// of that many chunks: 4 to 16 rows per workgroup).  16 waves a CU hide each other's loads, reductions and
// stores: 73920 x 5120 fp32 to bf16 takes 0.44 ms = 5.2 TB/s, with the next row's loads issued ahead
// 0.54 ms, and with more workgroups 0.48 to 0.55 ms.  Only rows past 8192 elements (AHEAD), of which a CU holds one
// at a time, load the next row ahead (8000 x 16384 fp32: 195 us, 215 without).
template <typename TX, typename TY, int NV, int LANES, bool AHEAD>
__global__ __launch_bounds__(MAXT) void layer_norm_fwd_kernel(
    const TX* __restrict__ x, int64_t ldx, int64_t rows, int C, const void* __restrict__ w,
    const void* __restrict__ b, int wtype, float eps, TY* __restrict__ y, int64_t ldy,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int nw) {
  constexpr int N = CHUNK<TX>;
  __shared__ float red[2][3 * MAXW];
  const int T = nw * 64, per = nw == 1 ? NARROW / LANES : 1;
  const int t = nw == 1 ? threadIdx.x & (LANES - 1) : threadIdx.x;
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
  int64_t row = (int64_t)blockIdx.x * per + (nw == 1 ? threadIdx.x / LANES : 0);
  const int64_t stride = (int64_t)gridDim.x * per;
  typename Raw<TX, N>::vec xr[NV];
  auto load = [&](int64_t r) {
    if (r < rows) {
#pragma unroll
      for (int j = 0; j < NV; ++j) xr[j] = load_raw<TX, N>(x + r * ldx + (t + j * T) * N, cnt[j]);
    }
  };
  if (AHEAD) load(row);
  for (int it = 0; row < rows; row += stride, ++it) {
    if (!AHEAD) load(row);
    float v[NV][N], mean, rstd;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) v[j][i] = (float)xr[j][i];
    if (AHEAD) load(row + stride);
    row_stats<NV, N, LANES>(v, cnt, C, nw, wave_n, eps, red[it & 1], mean, rstd);
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
// (part_w / part_b [gridDim.x][C]).  The sums take as many registers as a row, so 12 waves at most share a CU
// and the next row's loads are issued ahead: 32760 x 5120 bf16 takes 0.20 ms = 4.9 TB/s (0.46 without)
// (rows past 8192 elements, TMAX 1024: two registers sets of a row do not fit, each row is loaded when
// its turn comes).
template <typename TX, typename TY, int NV, int LANES, int TMAX>
__global__ __launch_bounds__(TMAX) void layer_norm_bwd_kernel(
    const TY* __restrict__ dy, int64_t lddy, const TX* __restrict__ x, int64_t ldx,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, int64_t rows, int C,
    const void* __restrict__ w, int wtype, TX* __restrict__ dx, int64_t lddx,
    float* __restrict__ part_w, float* __restrict__ part_b, int nw) {
  constexpr int N = CHUNK<TX>;
  __shared__ float red[2][2 * MAXW];
  __shared__ float join[NARROW * N];
  constexpr bool AHEAD = TMAX < MAXT;
  constexpr int GROUPS = NARROW / LANES;           // rows at a time with nw == 1
  const int T = nw * 64, per = nw == 1 ? GROUPS : 1;
  const int t = nw == 1 ? threadIdx.x & (LANES - 1) : threadIdx.x, wv_id = threadIdx.x >> 6;
  const int group = threadIdx.x / LANES;
  int cnt[NV];
  float wv[NV][N], sw[NV][N], sb[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    cnt[j] = min(max(C - (t + j * T) * N, 0), N);
#pragma unroll
    for (int i = 0; i < N; ++i) wv[j][i] = 1.f, sw[j][i] = 0.f, sb[j][i] = 0.f;
    if (w) load_any<N>(w, wtype, (int64_t)(t + j * T) * N, cnt[j], wv[j]);
  }
  int64_t row = (int64_t)blockIdx.x * per + (nw == 1 ? group : 0);
  const int64_t stride = (int64_t)gridDim.x * per;
  typename Raw<TX, N>::vec xr[NV];
  typename Raw<TY, N>::vec gr[NV];
  float mean_next = 0.f, rstd_next = 0.f;
  auto load = [&](int64_t r) {
    if (r < rows) {
      mean_next = mean_in[r];
      rstd_next = rstd_in[r];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        xr[j] = load_raw<TX, N>(x + r * ldx + (t + j * T) * N, cnt[j]);
        gr[j] = load_raw<TY, N>(dy + r * lddy + (t + j * T) * N, cnt[j]);
      }
    }
  };
  if (AHEAD) load(row);
  for (int it = 0; row < rows; row += stride, ++it) {
    if (!AHEAD) load(row);
    const float mean = mean_next, rstd = rstd_next;
    float xh[NV][N], g[NV][N], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        xh[j][i] = (float)xr[j][i];
        g[j][i] = (float)gr[j][i];
      }
    if (AHEAD) load(row + stride);
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
    s1 = row_sum<LANES>(s1);
    s2 = row_sum<LANES>(s2);
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
  // with nw == 1 the row groups of a workgroup hold the same columns: the first adds them in order
  auto put = [&](float* part, float (&s)[NV][N]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (nw == 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) join[i * NARROW + threadIdx.x] = s[j][i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
          s[j][i] = join[i * NARROW + t];
          for (int g = 1; g < GROUPS; ++g) s[j][i] += join[i * NARROW + g * LANES + t];
        }
      }
      if (nw > 1 || group == 0)
        store_n<float, N>(part + (int64_t)blockIdx.x * C + (t + j * T) * N, cnt[j], s[j]);
    }
  };
  if (part_w) put(part_w, sw);
  if (part_b) put(part_b, sb);
}

// out[c] = sum over p of part[p][c] for up to two [P][C] matrices (blockIdx.y): 16 columns per
// workgroup, every 64th row per group of 16 lanes, joined in a fixed order.
__global__ __launch_bounds__(1024) void layer_norm_dw_kernel(const float* __restrict__ part0,
                                                             const float* __restrict__ part1, int P,
                                                             int C, float* __restrict__ out0,
                                                             float* __restrict__ out1) {
  __shared__ float red[64][17];
  const float* part = blockIdx.y ? part1 : part0;
  float* out = blockIdx.y ? out1 : out0;
  if (!part) return;
  const int l = threadIdx.x & 15, g = threadIdx.x >> 4, c = blockIdx.x * 16 + l;
  float s = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int p = g; p < P; p += 64) s += part[(int64_t)p * C + c];
  }
  red[g][l] = s;
  __syncthreads();
  if (threadIdx.x < 256) {
    s = red[g * 4][l] + red[g * 4 + 1][l] + red[g * 4 + 2][l] + red[g * 4 + 3][l];
  }
  __syncthreads();
  if (threadIdx.x < 256) red[g][l] = s;
  __syncthreads();
  if (g == 0 && c < C) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += red[i][l];
    out[c] = s;
  }
}

// chunks per thread, lanes and waves for a row of C elements, at most 16 elements a thread
struct Split {
  int nv, lanes, nw;
  int64_t rows_at_once() const { return nw == 1 ? NARROW / lanes : 1; }
  int threads() const { return nw == 1 ? NARROW : nw * 64; }
};
// wide: threads a row may take before they take more than one chunk each.  The forward is fastest with few
// waves a row (40000 x 2048 bf16: 62 us with 2 waves, 94 with 4), the backward with more, for its registers
// (fp32 32760 x 1280: 92 us with 5 waves, 105 with 2).
constexpr int FWD_WIDE = 128, BWD_WIDE = 512;
Split split_for(int C, int x_type, int wide) {
  const int n = x_type ? 8 : 4, most = 16 / n, chunks = (C + n - 1) / n;
  int nv = 1;
  while (nv < most && chunks > wide * nv) ++nv;
  return {nv, chunks <= 16 ? 16 : chunks <= 32 ? 32 : 64, (chunks + 64 * nv - 1) / (64 * nv)};
}
// workgroups that share the CUs evenly, `waves` waves a CU
int grid_for_rows(int64_t rows, const Split& s, int waves) {
  const int64_t g = (rows + s.rows_at_once() - 1) / s.rows_at_once();
  const int each = waves / (s.threads() / 64), most = 256 * (each < 1 ? 1 : each);
  return (int)(g < most ? g : most);
}
constexpr int FWD_WAVES = 16, FWD_NARROW_WAVES = 24, BWD_WAVES = 12;
// The backward's workgroups each leave C partial sums: 256 of them (one a CU), and more where each still has
// four turns (1003 x 1021 fp16: 13 us in 256 workgroups, 18 in 1003).
int bwd_grid(int64_t rows, const Split& s) {
  if (!rows) return 0;
  const int g = grid_for_rows(rows, s, BWD_WAVES);
  const int64_t turns = (rows + 4 * s.rows_at_once() - 1) / (4 * s.rows_at_once());
  return g <= 256 || turns >= g ? g : (int)(turns > 256 ? turns : 256);
}

template <typename F>
void by_types(int xt, int yt, F f) {               // f(null pointers of the two types)
  const float* a = nullptr;
  const bf16* b = nullptr;
  const _Float16* h = nullptr;
  auto second = [&](auto* x) {
    if (yt == 0) f(x, a);
    else if (yt == 1) f(x, b);
    else f(x, h);
  };
  if (xt == 0) second(a);
  else if (xt == 1) second(b);
  else second(h);
}
template <int N>
using Int = std::integral_constant<int, N>;
template <int MOST, typename F>
void by_split(const Split& s, F f) {              // f(chunks per thread, lanes)
  if (s.nv == 1 && s.lanes == 16) f(Int<1>(), Int<16>());
  else if (s.nv == 1 && s.lanes == 32) f(Int<1>(), Int<32>());
  else if (s.nv == 1) f(Int<1>(), Int<64>());
  else if (s.nv == 2) f(Int<2>(), Int<64>());
  else if constexpr (MOST > 2) {
    if (s.nv == 3) f(Int<3>(), Int<64>());
    else f(Int<4>(), Int<64>());
  }
}
bool bad(int64_t rows, int64_t C, int xt, int yt, int wt) {
  return rows < 0 || C < 1 || C > MAXC || xt < 0 || xt > 2 || yt < 0 || yt > 2 || wt < 0 || wt > 2;
}
}  // namespace

extern "C" int64_t prfl_layer_norm_parts(int64_t rows, int64_t C, int x_type) {
  if (bad(rows, C, x_type, 0, 0)) return 0;
  return bwd_grid(rows, split_for((int)C, x_type, BWD_WIDE));
}

extern "C" int prfl_layer_norm_fwd(const void* x, int x_type, int64_t ldx, int64_t rows, int64_t C,
                                   const void* w, const void* b, int w_type, float eps, void* y,
                                   int y_type, int64_t ldy, float* mean, float* rstd, void* stream) {
  if (bad(rows, C, x_type, y_type, w_type) || (rows > 1 && (ldx < 0 || ldy < C)) || !(eps >= 0.f))
    return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  if (!x || !y || !mean || !rstd) return (int)hipErrorInvalidValue;
  hipStream_t s = (hipStream_t)stream;
  const Split sp = split_for((int)C, x_type, FWD_WIDE);
  const int grid = grid_for_rows(rows, sp, sp.nw == 1 ? FWD_NARROW_WAVES : FWD_WAVES);
  prfl_prof::begin(KID_LN, s);
  by_types(x_type, y_type, [&](auto* tx, auto* ty) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(tx)>>;
    using TY = std::remove_const_t<std::remove_pointer_t<decltype(ty)>>;
    by_split<16 / CHUNK<TX>>(sp, [&](auto nv, auto lanes) {
      auto kernel = layer_norm_fwd_kernel<TX, TY, nv(), lanes(), false>;
      if constexpr (nv() * CHUNK<TX> == 16)      // rows past 8192 elements: more than 8 waves
        if (sp.nw > 8) kernel = layer_norm_fwd_kernel<TX, TY, nv(), lanes(), true>;
      hipLaunchKernelGGL(kernel, dim3(grid), dim3(sp.threads()), 0, s, (const TX*)x, ldx, rows, (int)C, w, b,
                         w_type, eps, (TY*)y, ldy, mean, rstd, sp.nw);
    });
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
      ((dw || db) && !part) || (rows && (dx || dw || db) && (!dy || !x || !mean || !rstd)))
    return (int)hipErrorInvalidValue;
  hipStream_t s = (hipStream_t)stream;
  const Split sp = split_for((int)C, x_type, BWD_WIDE);
  const int grid = bwd_grid(rows, sp);
  float* pw = dw ? part : nullptr;
  float* pb = db ? part + (dw ? (int64_t)grid * C : 0) : nullptr;
  prfl_prof::begin(KID_LN, s);
  if (rows && (dx || dw || db)) {
    by_types(x_type, y_type, [&](auto* tx, auto* ty) {
      using TX = std::remove_const_t<std::remove_pointer_t<decltype(tx)>>;
      using TY = std::remove_const_t<std::remove_pointer_t<decltype(ty)>>;
      by_split<16 / CHUNK<TX>>(sp, [&](auto nv, auto lanes) {
        auto kernel = layer_norm_bwd_kernel<TX, TY, nv(), lanes(), 512>;
        if constexpr (nv() * CHUNK<TX> == 16)      // rows past 8192 elements: more than 8 waves
          if (sp.nw > 8) kernel = layer_norm_bwd_kernel<TX, TY, nv(), lanes(), MAXT>;
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(sp.threads()), 0, s,
                           (const TY*)dy, lddy, (const TX*)x, ldx, mean, rstd, rows, (int)C, w, w_type,
                           (TX*)dx, lddx, pw, pb, sp.nw);
      });
    });
  }
  if (dw || db)
    hipLaunchKernelGGL(layer_norm_dw_kernel, dim3((C + 15) / 16, 2), dim3(1024), 0, s, pw, pb, grid,
                       (int)C, dw, db);
  prfl_prof::set_work((double)rows * C * (2 * (x_type ? 2 : 4) + (y_type ? 2 : 4)));
  prfl_prof::end(KID_LN, s);
  PRFL_LAUNCH_CHECK();
  return 0;
}
