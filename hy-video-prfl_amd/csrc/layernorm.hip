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

// A lane's N columns start at `at`: its stripe's, or where the row ends inside or before that the row's last N
// (negative in rows narrower than N).  Columns i < lo of them are another lane's (lo >= N: all of them); they
// count as zeros and are not stored.  So every load is one whole vector inside the row: a lane that loaded its last
// elements one by one into the same registers would first wait for the vectors that the other lanes
// have under way, the next row's among them (backward of 20651 x 6080 bf16: 259 us so, 164 with whole vectors).
struct Own {
  int at, lo;
};
template <int N>
__device__ __forceinline__ Own own_columns(int column, int C) {
  const int at = min(column, C - N);
  return {at, column - at};
}
template <typename T, int N, bool SHORT>
__device__ __forceinline__ typename Raw<T, N>::vec load_raw(const T* row, const Own& o, int C) {
  typename Raw<T, N>::vec t;
  if (!SHORT || C >= N) {
    t = *(const typename Raw<T, N>::at*)(row + o.at);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = i >= o.lo ? row[o.at + i] : (T)0.f;
  }
  return t;
}
template <bool SHORT, typename T, int N>
__device__ __forceinline__ void store_n(T* row, const Own& o, int C, const float (&v)[N]) {
  if (!SHORT || C >= N) {
    typename Raw<T, N>::vec t;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = (T)v[i];
    if (o.lo < N) *(typename Raw<T, N>::at*)(row + o.at) = t;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i >= o.lo) row[o.at + i] = (T)v[i];
  }
}
template <int NV, int N>
__device__ __forceinline__ bool any_not_own(const Own (&own)[NV]) {
  bool some = false;
#pragma unroll
  for (int j = 0; j < NV; ++j) some |= own[j].lo > 0;
  return __any(some);
}
template <int N, bool SHORT>
__device__ __forceinline__ void load_any(const void* p, int type, const Own& o, int C, float (&v)[N]) {
  auto widen = [&](auto raw) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)raw[i];
  };
  if (type == 0) widen(load_raw<float, N, SHORT>((const float*)p, o, C));
  else if (type == 1) widen(load_raw<bf16, N, SHORT>((const bf16*)p, o, C));
  else widen(load_raw<_Float16, N, SHORT>((const _Float16*)p, o, C));
}

// mean and rstd of a row held as v[NV][N] per thread.  Within a wave two passes over the
// registers; across waves the partial sums of squares about the waves' own means are joined:
//   M2 = sum_w M2_w + n_w (mu_w - mu)^2,
// so a mean far from zero costs no digits.  red: the row's sums per wave, double-buffered by the caller so
// that one barrier a row is enough; every 16 lanes join them for themselves.  Sums over lanes go by DPP and
// lane swaps, not through LDS: a row's turn is a chain of them (32760 x 5120 bf16 forward: 130 us, 147 with
// shuffles and a loop over the waves).
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
  v = add_dpp<0xb1>(v);            // quad_perm 1 0 3 2
  v = add_dpp<0x4e>(v);            // quad_perm 2 3 0 1
  v = add_dpp<0x141>(v);           // row_half_mirror
  v = add_dpp<0x140>(v);           // row_mirror
  if constexpr (LANES >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if constexpr (LANES == 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return v;
}
template <int NV, int N, int LANES>
__device__ __forceinline__ void row_stats(const float (&v)[NV][N], const Own (&own)[NV], bool ragged, int C, int nw,
                                          int wave_n, float eps, float* red, float& mean,
                                          float& rstd) {
  float s = 0.f;
  if (ragged) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) s += i >= own[j].lo ? v[j][i] : 0.f;
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) s += v[j][i];
  }
  s = row_sum<LANES>(s);
  const float mw = wave_n > 0 ? s / wave_n : 0.f;
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = i >= own[j].lo ? v[j][i] - mw : 0.f;
      q += d * d;
    }
  q = row_sum<LANES>(q);
  if (nw == 1) {
    mean = mw;
  } else {
    const int w = threadIdx.x >> 6, l = threadIdx.x & 15;
    if ((threadIdx.x & 63) == 0) {
      red[w] = s;
      red[MAXW + w] = q;
      red[2 * MAXW + w] = (float)wave_n;
    }
    __syncthreads();
    const bool some = l < nw;
    const float si = some ? red[l] : 0.f, qi = some ? red[MAXW + l] : 0.f, n = some ? red[2 * MAXW + l] : 0.f;
    mean = row_sum<16>(si) / C;
    const float d = n > 0.f ? si / n - mean : 0.f;
    q = row_sum<16>(qi + n * d * d);
  }
  rstd = 1.f / sqrtf(q / C + eps);
}

// One row per workgroup at a time (nw waves), or with nw == 1 per LANES lanes (64, or 32 / 16 for rows
// of that many chunks: 4 to 16 rows per workgroup).  16 waves a CU hide each other's loads, reductions and
// stores: 73920 x 5120 fp32 to bf16 takes 0.43 ms = 5.2 TB/s; with 24 waves a CU 0.46 ms, with the next row's loads
// issued ahead 0.47 ms (8000 x 16384 fp32: 184 us, 200 with them).
template <typename TX, typename TY, int NV, int LANES>
__global__ __launch_bounds__(MAXT) void layer_norm_fwd_kernel(
    const TX* __restrict__ x, int64_t ldx, int64_t rows, int C, const void* __restrict__ w,
    const void* __restrict__ b, int wtype, float eps, TY* __restrict__ y, int64_t ldy,
    float* __restrict__ mean_out, float* __restrict__ rstd_out, int nw) {
  constexpr int N = CHUNK<TX>;
  __shared__ float red[2][3 * MAXW];
  const int T = nw * 64, per = nw == 1 ? NARROW / LANES : 1;
  const int t = nw == 1 ? threadIdx.x & (LANES - 1) : threadIdx.x;
  const int first = t & ~63;                       // the wave's first chunk in each stripe
  Own own[NV];
  int wave_n = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    own[j] = own_columns<N>((t + j * T) * N, C);
    wave_n += min(max(C - (first + j * T) * N, 0), 64 * N);
  }
  float wv[NV][N], bv[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < N; ++i) wv[j][i] = 1.f, bv[j][i] = 0.f;
    if (w) load_any<N, LANES == 16>(w, wtype, own[j], C, wv[j]);
    if (b) load_any<N, LANES == 16>(b, wtype, own[j], C, bv[j]);
  }
  int64_t row = (int64_t)blockIdx.x * per + (nw == 1 ? threadIdx.x / LANES : 0);
  const int64_t stride = (int64_t)gridDim.x * per;
  const bool ragged = any_not_own<NV, N>(own);
  typename Raw<TX, N>::vec xr[NV];
  for (int it = 0; row < rows; row += stride, ++it) {
    float v[NV][N], mean, rstd;
#pragma unroll
    for (int j = 0; j < NV; ++j) xr[j] = load_raw<TX, N, LANES == 16>(x + row * ldx, own[j], C);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) v[j][i] = (float)xr[j][i];
    row_stats<NV, N, LANES>(v, own, ragged, C, nw, wave_n, eps, red[it & 1], mean, rstd);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float o[N];
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fmaf((v[j][i] - mean) * rstd, wv[j][i], bv[j][i]);
      store_n<LANES == 16, TY, N>(y + row * ldy, own[j], C, o);
    }
    if (t == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

// dx of each row and, where asked for, the workgroup's sums of dy xhat and dy over its rows
// (part_w / part_b [gridDim.x][C]).  The sums take as many registers as a row, so 12 waves at most share a CU
// and the next row's loads are issued ahead: 32760 x 5120 bf16 takes 0.18 ms = 5.6 TB/s (0.28 without)
// (rows past 8192 elements, TMAX 1024: 128 registers hold one set of a row, which is loaded when its turn comes, and
// where x or dy is 32 bits wide or dy is fp16 not all of that: 2 to 26 registers go to scratch.  8000 x 16384 all the same: fp32
// 319 us = 4.9 TB/s, fp32 with fp16 dy 308 = 4.3, bf16 163 = 4.8, fp16 164 = 4.8).
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
  Own own[NV];
  float wv[NV][N], sw[NV][N], sb[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    own[j] = own_columns<N>((t + j * T) * N, C);
#pragma unroll
    for (int i = 0; i < N; ++i) wv[j][i] = 1.f, sw[j][i] = 0.f, sb[j][i] = 0.f;
    if (w) load_any<N, LANES == 16>(w, wtype, own[j], C, wv[j]);
  }
  int64_t row = (int64_t)blockIdx.x * per + (nw == 1 ? group : 0);
  const int64_t stride = (int64_t)gridDim.x * per;
  const bool ragged = any_not_own<NV, N>(own);
  typename Raw<TX, N>::vec xr[NV];
  typename Raw<TY, N>::vec gr[NV];
  float mean_next = 0.f, rstd_next = 0.f;
  auto load = [&](int64_t r) {
    if (r < rows) {
      mean_next = mean_in[r];
      rstd_next = rstd_in[r];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        xr[j] = load_raw<TX, N, LANES == 16>(x + r * ldx, own[j], C);
        gr[j] = load_raw<TY, N, LANES == 16>(dy + r * lddy, own[j], C);
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
      }
    if (ragged) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          s1 += i >= own[j].lo ? g[j][i] : 0.f;
          s2 += i >= own[j].lo ? g[j][i] * xh[j][i] : 0.f;
        }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          s1 += g[j][i];
          s2 = fmaf(g[j][i], xh[j][i], s2);
        }
    }
    s1 = row_sum<LANES>(s1);
    s2 = row_sum<LANES>(s2);
    if (nw > 1) {
      float* r = red[it & 1];
      if ((threadIdx.x & 63) == 0) r[wv_id] = s1, r[MAXW + wv_id] = s2;
      __syncthreads();
      const int l = threadIdx.x & 15;
      s1 = row_sum<16>(l < nw ? r[l] : 0.f);
      s2 = row_sum<16>(l < nw ? r[MAXW + l] : 0.f);
    }
    const float m1 = s1 / C, m2 = s2 / C;
    if (dx) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float o[N];
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = rstd * (g[j][i] - m1 - xh[j][i] * m2);
        store_n<LANES == 16, TX, N>(dx + row * lddx, own[j], C, o);
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
        store_n<LANES == 16, float, N>(part + (int64_t)blockIdx.x * C, own[j], C, s[j]);
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
// wide: lanes a row may take before they take more than one chunk each.  The forward is fastest with one wave a
// row where that holds it (60000 x 640 bf16: 27 us, 47 with two waves; 37117 x 592 fp32: 22 and 30).  So is the backward up
// to three chunks a lane (60000 x 640 bf16: 44 us, 58 with two waves; 37117 x 592 fp32: 41 and 45); rows past that take
// more waves, for its registers (32760 x 1280 fp32: 92 us with 5 waves, 98 with 2).
constexpr int FWD_WIDE = 64, BWD_WIDE = 512;
Split split_for(int C, int x_type, bool backward) {
  const int n = x_type ? 8 : 4, most = 16 / n, chunks = (C + n - 1) / n;
  const int wide = !backward || chunks <= 64 * (most < 3 ? most : 3) ? FWD_WIDE : BWD_WIDE;
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
constexpr int FWD_WAVES = 16, FWD_NARROW_WAVES = 24, BWD_WAVES = 12, BWD_WIDE_WAVES = 8;
// The backward's rows of several waves and chunks are fastest with one workgroup a CU (20651 x 6080 bf16: 142 us, 155
// with two), the others with 12 waves (37117 x 592 fp32: 45 us, 63 with 8).  Its workgroups each leave C partial
// sums: 128 of them, and more where each still has four turns (300 x 16384 bf16: 22.5 us in 128 workgroups, 27.6 in
// 256; 400 x 5120: 14.6 and 18.0; 4000 x 256: 8.4, 7.9 in 256, 9.4 in 500).  Up to four turns go to a single
// workgroup, whose sums are dw and db: one launch less.
int bwd_grid(int64_t rows, const Split& s) {
  if (!rows) return 0;
  if (rows <= 4 * s.rows_at_once()) return 1;
  const int g = grid_for_rows(rows, s, s.nv > 1 && s.nw > 1 ? BWD_WIDE_WAVES : BWD_WAVES);
  const int64_t turns = (rows + 4 * s.rows_at_once() - 1) / (4 * s.rows_at_once());
  return g <= 128 || turns >= g ? g : (int)(turns > 128 ? turns : 128);
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
  const int grid = bwd_grid(rows, split_for((int)C, x_type, true));
  return grid > 1 ? grid : 0;
}

extern "C" int prfl_layer_norm_fwd(const void* x, int x_type, int64_t ldx, int64_t rows, int64_t C,
                                   const void* w, const void* b, int w_type, float eps, void* y,
                                   int y_type, int64_t ldy, float* mean, float* rstd, void* stream) {
  if (bad(rows, C, x_type, y_type, w_type) || (rows > 1 && (ldx < 0 || ldy < C)) || !(eps >= 0.f))
    return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  if (!x || !y || !mean || !rstd) return (int)hipErrorInvalidValue;
  hipStream_t s = (hipStream_t)stream;
  const Split sp = split_for((int)C, x_type, false);
  const int grid = grid_for_rows(rows, sp, sp.nw == 1 ? FWD_NARROW_WAVES : FWD_WAVES);
  prfl_prof::begin(KID_LN, s);
  by_types(x_type, y_type, [&](auto* tx, auto* ty) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(tx)>>;
    using TY = std::remove_const_t<std::remove_pointer_t<decltype(ty)>>;
    by_split<16 / CHUNK<TX>>(sp, [&](auto nv, auto lanes) {
      hipLaunchKernelGGL((layer_norm_fwd_kernel<TX, TY, nv(), lanes()>), dim3(grid), dim3(sp.threads()), 0, s,
                         (const TX*)x, ldx, rows, (int)C, w, b, w_type, eps, (TY*)y, ldy, mean, rstd, sp.nw);
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
      (rows && (dx || dw || db) && (!dy || !x || !mean || !rstd)))
    return (int)hipErrorInvalidValue;
  hipStream_t s = (hipStream_t)stream;
  const Split sp = split_for((int)C, x_type, true);
  const int grid = bwd_grid(rows, sp);
  if (grid > 1 && (dw || db) && !part) return (int)hipErrorInvalidValue;
  float* pw = grid <= 1 || !dw ? dw : part;
  float* pb = grid <= 1 || !db ? db : part + (dw ? (int64_t)grid * C : 0);
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
  if (grid != 1 && (dw || db))
    hipLaunchKernelGGL(layer_norm_dw_kernel, dim3((C + 15) / 16, 2), dim3(1024), 0, s, pw, pb, grid,
                       (int)C, dw, db);
  prfl_prof::set_work((double)rows * C * (2 * (x_type ? 2 : 4) + (y_type ? 2 : 4)));
  prfl_prof::end(KID_LN, s);
  PRFL_LAUNCH_CHECK();
  return 0;
}
