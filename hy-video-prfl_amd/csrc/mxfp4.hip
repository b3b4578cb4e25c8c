// Microscaled four-bit floating point (OCP MX, e2m1 elements with one e8m0 scale per 32 elements
// of a row): quantisation, reading back, and the product y = x W^T + b on the block-scaled MFMA.
//
//   e    = floor(log2(max |v|)) - 2 over the 32, at least -127   (0 for an all-zero block: -127)
//   code = v / 2^e rounded to the nearest of 0 .5 1 1.5 2 3 4 6, ties to the even code, at most 6
//   a block with a NaN or an infinity has the scale 0xff: all its 32 values read back as NaN.
//
// Layout ("tiled"): the matrix in pieces of 64 rows x 128 columns, row pieces outermost; a piece is
// four MFMA operands [row half][column half][lane][16 B], lane = 32 * block + row: the 32 codes
// of one block, low nibble first.  The scales of a piece are [lane][4]: one byte for each of the
// piece's four operands, so that one dword a lane holds all that its four MFMAs take (opsel
// picks the byte).  Every operand is then one contiguous KiB in lane order, from HBM to the
// registers, and a lane's 16 bytes are exactly one block.  Rows and columns of the padding (to 64
// and 128) are zeros.
#include "common.h"

namespace {
typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

constexpr int NT = 256;
constexpr int PIECE = 4096, PIECE_S = 256;        // bytes of a piece: codes, scales

template <typename T, int N>
struct Loaded {
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec at __attribute__((aligned(sizeof(T))));
};

// 8 codes of v[8] / 2^(scale - 127)
__device__ __forceinline__ uint32_t pack8(const float (&v)[8], float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}
// the e8m0 byte of a block whose largest magnitude has these bits; 2^(byte - 127)
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;              // 0 for zero and subnormals
  return e == 255 ? 255u : (e > 2 ? e - 2 : 0u);
}
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}

// One workgroup per piece.  A quad of lanes has one block, 8 elements a lane; a wave has 8 rows x 2
// blocks at a time, so that it reads and writes runs of 128 bytes or more.
template <typename T>
__global__ __launch_bounds__(NT) void quant_kernel(const T* __restrict__ x, int64_t ldx, int64_t M,
                                                   int K, int steps, uint8_t* __restrict__ q,
                                                   uint8_t* __restrict__ s) {
  __shared__ uint8_t sc[PIECE_S];
  const int64_t piece = blockIdx.x, g = piece / steps;
  const int k0 = (int)(piece - g * steps) * 128;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int r8 = lane >> 3, blk = (lane >> 2) & 1, part = lane & 3;
  float v[4][8];
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int task = wid * 4 + it, kh = task & 1, row = (task >> 1) * 8 + r8;
    const int k = k0 + kh * 64 + blk * 32 + part * 8;
    const int64_t m = g * 64 + row;
    const int n = m < M ? min(K - k, 8) : 0;
    const T* p = x + m * ldx + k;
    if (n >= 8) {
      const typename Loaded<T, 8>::vec t = *(const typename Loaded<T, 8>::at*)p;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[it][i] = (float)t[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[it][i] = i < n ? (float)p[i] : 0.f;
    }
  }
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int task = wid * 4 + it, kh = task & 1, row = (task >> 1) * 8 + r8;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[it][i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
    const uint32_t byte = scale_byte(top);
    const uint32_t w = byte == 255 ? 0u : pack8(v[it], scale_value(byte));
    const int unit = (row >> 5) * 2 + kh, l = blk * 32 + (row & 31);
    *(uint32_t*)(q + piece * PIECE + unit * 1024 + l * 16 + part * 4) = w;
    if (part == 0) sc[l * 4 + unit] = (uint8_t)byte;
  }
  __syncthreads();
  if (threadIdx.x < 64)
    *(uint32_t*)(s + piece * PIECE_S + threadIdx.x * 4) = *(const uint32_t*)(sc + threadIdx.x * 4);
}

// codes and scales back to values, row-major (exact in bf16 and fp32 for what quant_kernel wrote)
template <typename T>
__global__ __launch_bounds__(NT) void dequant_kernel(const uint8_t* __restrict__ q,
                                                     const uint8_t* __restrict__ s, int64_t M, int K,
                                                     int steps, T* __restrict__ out, int64_t ldo) {
  const int64_t piece = blockIdx.x, g = piece / steps;
  const int k0 = (int)(piece - g * steps) * 128;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int r8 = lane >> 3, blk = (lane >> 2) & 1, part = lane & 3;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int task = wid * 4 + it, kh = task & 1, row = (task >> 1) * 8 + r8;
    const int k = k0 + kh * 64 + blk * 32 + part * 8;
    const int64_t m = g * 64 + row;
    if (m >= M || k >= K) continue;
    const int unit = (row >> 5) * 2 + kh, l = blk * 32 + (row & 31);
    const uint32_t w = *(const uint32_t*)(q + piece * PIECE + unit * 1024 + l * 16 + part * 4);
    const float sv = scale_value(s[piece * PIECE_S + l * 4 + unit]);
    float v[8];
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
    T* p = out + m * ldo + k;
    if (K - k >= 8) {
      typename Loaded<T, 8>::vec t;
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = (T)(v[i] * sv);
      *(typename Loaded<T, 8>::at*)p = t;
    } else {
      for (int i = 0; i < K - k; ++i) p[i] = (T)(v[i] * sv);
    }
  }
}

// ---------------------------------------------------------------------------------- product --
// D (32 x 32) += A B^T of one operand pair, 64 deep; OA / OB: the byte of the lane's scale dword.
template <int OA, int OB>
__device__ __forceinline__ f32x16 mfma4(u32x4 a, u32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
  const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, OA, (int)sa, OB, (int)sb);
}

struct MxArgs {
  const uint8_t* wq;      // W [N][K] tiled
  const uint8_t* ws;
  const uint8_t* xq;      // x [M][K] tiled
  const uint8_t* xs;
  const bf16* bias;       // [N] or null
  bf16* y;
  int64_t ldy;
  int64_t M;
  int N, steps;
};

// W is the MFMA's first operand, so a lane holds four consecutive columns n of one row m at a
// time: register r of tile (i, j) is n = 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4, m = 32 j + lane % 32
__device__ __forceinline__ void store4(const MxArgs& a, int64_t m, int n, const float (&v)[4]) {
  if (m >= a.M) return;
  bf16* p = a.y + m * a.ldy + n;
  if (n + 4 <= a.N) {
    typename Loaded<bf16, 4>::vec t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = f2bf(v[i] + (a.bias ? bf2f(a.bias[n + i]) : 0.f));
    *(typename Loaded<bf16, 4>::at*)p = t;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) p[i] = f2bf(v[i] + (a.bias ? bf2f(a.bias[n + i]) : 0.f));
  }
}

// 64 columns x 64 rows of y per wave, the operands straight from memory
__global__ __launch_bounds__(NT) void mx_gemm_kernel(MxArgs a) {
  const int lane = threadIdx.x & 63;
  const int gn = (a.N + 63) / 64;
  const int64_t gm = (a.M + 63) / 64, unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= gn * gm) return;
  const int64_t n = unit % gn, m = unit / gn;
  const u32x4* w = (const u32x4*)(a.wq + n * a.steps * PIECE) + lane;
  const u32x4* x = (const u32x4*)(a.xq + m * a.steps * PIECE) + lane;
  const uint32_t* sw = (const uint32_t*)(a.ws + n * a.steps * PIECE_S) + lane;
  const uint32_t* sx = (const uint32_t*)(a.xs + m * a.steps * PIECE_S) + lane;
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = (f32x16)(0.f);
  for (int k = 0; k < a.steps; ++k) {
    u32x4 wv[4], xv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      wv[u] = w[k * 256 + u * 64];
      xv[u] = x[k * 256 + u * 64];
    }
    const uint32_t s0 = sw[k * 64], s1 = sx[k * 64];
    acc[0][0] = mfma4<0, 0>(wv[0], xv[0], acc[0][0], s0, s1);
    acc[0][1] = mfma4<0, 2>(wv[0], xv[2], acc[0][1], s0, s1);
    acc[1][0] = mfma4<2, 0>(wv[2], xv[0], acc[1][0], s0, s1);
    acc[1][1] = mfma4<2, 2>(wv[2], xv[2], acc[1][1], s0, s1);
    acc[0][0] = mfma4<1, 1>(wv[1], xv[1], acc[0][0], s0, s1);
    acc[0][1] = mfma4<1, 3>(wv[1], xv[3], acc[0][1], s0, s1);
    acc[1][0] = mfma4<3, 1>(wv[3], xv[1], acc[1][0], s0, s1);
    acc[1][1] = mfma4<3, 3>(wv[3], xv[3], acc[1][1], s0, s1);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v[4] = {acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
        store4(a, m * 64 + j * 32 + (lane & 31), (int)n * 64 + i * 32 + 8 * r + 4 * (lane >> 5), v);
      }
}

bool too_large(int64_t rows, int64_t cols) {       // pieces are counted in 31 bits
  return rows < 0 || cols < 1 || cols > (1 << 24) ||
         ((rows + 63) / 64) * ((cols + 127) / 128) > 0x7fffffff;
}
}  // namespace

extern "C" int prfl_quant_mxfp4(const void* x, int x_type, int64_t ldx, int64_t M, int64_t K, void* q,
                                void* s, void* stream) {
  if (too_large(M, K) || x_type < 0 || x_type > 2 || (M > 1 && ldx < 0)) return (int)hipErrorInvalidValue;
  if (M == 0) return 0;
  if (!x || !q || !s || ((uintptr_t)q & 15) || ((uintptr_t)s & 3)) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  const int steps = (int)((K + 127) / 128);
  const dim3 grid((unsigned)((M + 63) / 64 * steps));
  prfl_prof::begin(KID_ELTWISE, st);
  if (x_type == 0)
    hipLaunchKernelGGL(quant_kernel<float>, grid, dim3(NT), 0, st, (const float*)x, ldx, M, (int)K, steps,
                       (uint8_t*)q, (uint8_t*)s);
  else if (x_type == 1)
    hipLaunchKernelGGL(quant_kernel<bf16>, grid, dim3(NT), 0, st, (const bf16*)x, ldx, M, (int)K, steps,
                       (uint8_t*)q, (uint8_t*)s);
  else
    hipLaunchKernelGGL(quant_kernel<_Float16>, grid, dim3(NT), 0, st, (const _Float16*)x, ldx, M, (int)K,
                       steps, (uint8_t*)q, (uint8_t*)s);
  prfl_prof::set_work((double)M * K * (x_type ? 2.53125 : 4.53125));
  prfl_prof::end(KID_ELTWISE, st);
  PRFL_LAUNCH_CHECK();
  return 0;
}

extern "C" int prfl_dequant_mxfp4(const void* q, const void* s, int64_t M, int64_t K, void* out,
                                  int out_f32, int64_t ldo, void* stream) {
  if (too_large(M, K) || (M > 1 && ldo < K)) return (int)hipErrorInvalidValue;
  if (M == 0) return 0;
  if (!q || !s || !out || ((uintptr_t)q & 15) || ((uintptr_t)s & 3)) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  const int steps = (int)((K + 127) / 128);
  const dim3 grid((unsigned)((M + 63) / 64 * steps));
  if (out_f32)
    hipLaunchKernelGGL(dequant_kernel<float>, grid, dim3(NT), 0, st, (const uint8_t*)q, (const uint8_t*)s,
                       M, (int)K, steps, (float*)out, ldo);
  else
    hipLaunchKernelGGL(dequant_kernel<bf16>, grid, dim3(NT), 0, st, (const uint8_t*)q, (const uint8_t*)s,
                       M, (int)K, steps, (bf16*)out, ldo);
  PRFL_LAUNCH_CHECK();
  return 0;
}

extern "C" int prfl_gemm_mxfp4(const void* xq, const void* xs, const void* wq, const void* ws,
                               const void* bias, void* y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                               void* stream) {
  if (too_large(M, K) || too_large(N, K) || N < 1 || N > (1 << 24) || (M > 1 && ldy < N) ||
      ((M + 63) / 64) * ((N + 63) / 64) > 0x7fffffff)
    return (int)hipErrorInvalidValue;
  if (M == 0) return 0;
  if (!xq || !xs || !wq || !ws || !y || (((uintptr_t)xq | (uintptr_t)wq) & 15) ||
      (((uintptr_t)xs | (uintptr_t)ws) & 3))
    return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  MxArgs a{(const uint8_t*)wq, (const uint8_t*)ws, (const uint8_t*)xq, (const uint8_t*)xs,
           (const bf16*)bias, (bf16*)y, ldy, M, (int)N, (int)((K + 127) / 128)};
  const int64_t units = ((M + 63) / 64) * ((N + 63) / 64);
  prfl_prof::begin(KID_GEMM, st);
  hipLaunchKernelGGL(mx_gemm_kernel, dim3((unsigned)((units + 3) / 4)), dim3(NT), 0, st, a);
  prfl_prof::set_work(2.0 * M * N * K);
  prfl_prof::end(KID_GEMM, st);
  PRFL_LAUNCH_CHECK();
  return 0;
}
