// Microscaled four-bit floating point (OCP MX, e2m1 elements with one e8m0 scale per 32 elements
// of a row): quantisation, reading back, and the product y = x W^T + b on the block-scaled MFMA.
//
//   e    = floor(log2(max |v|)) - 2 over the 32, at least -127 (as for a block of zeros)
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
// time: register 4 q + c of a 32 x 32 tile is n = 8 q + 4 (lane / 32) + c, m = lane % 32

// tile of workgroup bid: every eighth workgroup runs on the same XCD, so XCD k gets the k-th eighth of
// the tiles, and within it 8 tile rows advance over the tile columns together (their operands
// meet in that XCD's L2)
__device__ __forceinline__ void tile_of(int bid, int ntm, int ntn, int& tm, int& tn) {
  const int all = ntm * ntn, xcd = bid & 7, q = all >> 3, r = all & 7;
  const int w = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
  const int g = w / (8 * ntn), rows = min(ntm - g * 8, 8), in = w - g * 8 * ntn;
  tm = g * 8 + in % rows;
  tn = in / rows;
}

// LDS-DMA of 4 B a lane (lane i lands at m0 + 4 i) from a buffer at voff + soff
__device__ __forceinline__ void dma4_step(i32x4 srd, uint32_t voff, uint32_t soff) {
  asm volatile("buffer_load_dword %0, %1, %2 offen lds"
               :: "v"(voff), "s"(srd), "s"(__builtin_amdgcn_readfirstlane(soff)) : "memory");
}

// Few rows, or few columns and a long K: 32 MT rows (MT 1 or 2; blockIdx.y) x 32 columns of y per workgroup, its
// 16 waves taking every 16th step of 128 along K, their partial sums joined through LDS in wave order.  W is
// read once per row group, in lane order, with up to four steps of it in flight per wave: the time is that of
// launch, first loads and the join (5120 x 5120, one round of workgroups: 4.5 us for 32 rows, 6.0 for 64).
// FUSED: x comes as it is, at most 32 rows and 1024 blocks of 32, and every workgroup quantises all of it, a
// block per thread, into LDS ([block][row]: rows beyond M take no room) -- one launch instead of two, while W's
// first loads are under way; else x comes tiled.
template <typename T, int N>
__device__ __forceinline__ void load_block(const T* p, int n, float (&v)[N]) {
#pragma unroll
  for (int c = 0; c < N; c += 8) {
    if (n >= c + 8) {
      const typename Loaded<T, 8>::vec t = *(const typename Loaded<T, 8>::at*)(p + c);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c + i] = (float)t[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c + i] = c + i < n ? (float)p[c + i] : 0.f;
    }
  }
}
constexpr int ROWS_WAVES = 16, ROWS_FUSED = 64 * ROWS_WAVES;

template <typename T, int MT, bool FUSED>
__global__ __launch_bounds__(64 * ROWS_WAVES) void mx_rows_kernel(MxArgs a, const T* __restrict__ x, int64_t ldx,
                                                                  int K) {
  __shared__ __attribute__((aligned(16))) float part[ROWS_WAVES * 1024];
  __shared__ __attribute__((aligned(16))) u32x4 lx[FUSED ? ROWS_FUSED : 1];
  __shared__ uint8_t lsx[FUSED ? ROWS_FUSED : 1];
  const int lane = threadIdx.x & 63, row = lane & 31, blk = lane >> 5;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nt = blockIdx.x, steps = a.steps;
  const int64_t g = blockIdx.y;                     // row piece
  const int M = (int)min(a.M - g * 64, (int64_t)64);
  const uint8_t* w = a.wq + (int64_t)(nt >> 1) * steps * PIECE + (nt & 1) * 2048 + lane * 16;
  const uint8_t* sw = a.ws + (int64_t)(nt >> 1) * steps * PIECE_S + lane * 4;
  constexpr int AHEAD = 4;
  f32x16 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = (f32x16)(0.f);

  u32x4 wv[AHEAD][2];
  uint32_t sv[AHEAD];
  auto load_w = [&](int k0) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = k0 + u * ROWS_WAVES;
      if (k >= steps) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) wv[u][h] = *(const u32x4*)(w + (int64_t)k * PIECE + h * 1024);
      sv[u] = *(const uint32_t*)(sw + (int64_t)k * PIECE_S) >> (16 * (nt & 1));
    }
  };
  load_w(wid);
  if constexpr (FUSED) {
    const int blocks = (K + 31) / 32, b = threadIdx.x / M, m = threadIdx.x - b * M;
    if (b < blocks) {
      float v[32];
      load_block(x + m * ldx + b * 32, K - b * 32, v);
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
      const uint32_t byte = scale_byte(top);
      u32x4 q;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e[8] = {v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3],
                            v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]};
        q[i] = byte == 255 ? 0u : pack8(e, scale_value(byte));
      }
      lx[b * M + m] = q;
      lsx[b * M + m] = (uint8_t)byte;
    }
    __syncthreads();
  }
  for (int k0 = wid; k0 < steps; k0 += AHEAD * ROWS_WAVES) {
    if (k0 != wid) load_w(k0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = k0 + u * ROWS_WAVES;
      if (k >= steps) break;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        u32x4 xv[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        uint32_t sx = 0;
        if constexpr (FUSED) {
          const int blocks = (K + 31) / 32;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int b = k * 4 + h * 2 + blk;
            if (row < M && b < blocks) {
              xv[h] = lx[b * M + row];
              sx |= (uint32_t)lsx[b * M + row] << (8 * h);
            }
          }
        } else if (m * 32 + row < M) {
          const uint8_t* xp = a.xq + (g * steps + k) * PIECE + m * 2048 + lane * 16;
          xv[0] = *(const u32x4*)xp;
          xv[1] = *(const u32x4*)(xp + 1024);
          sx = *(const uint32_t*)(a.xs + (g * steps + k) * PIECE_S + lane * 4) >> (16 * m);
        }
        acc[m] = mfma4<0, 0>(wv[u][0], xv[0], acc[m], sv[u], sx);
        acc[m] = mfma4<1, 1>(wv[u][1], xv[1], acc[m], sv[u], sx);
      }
    }
  }
  // register 4 q + c of lane l is column 8 q + 4 (l / 32) + c of row l % 32
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m) __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 v = {acc[m][4 * q], acc[m][4 * q + 1], acc[m][4 * q + 2], acc[m][4 * q + 3]};
      *(f32x4*)(part + wid * 1024 + q * 256 + lane * 4) = v;
    }
    __syncthreads();
    const int t = threadIdx.x, l = (t >> 2) & 63, mm = m * 32 + (l & 31);
    const int n = nt * 32 + 8 * (t >> 8) + 4 * (l >> 5) + (t & 3);
    if (mm < M && n < a.N) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < ROWS_WAVES; ++i) s += part[i * 1024 + t];
      a.y[(g * 64 + mm) * a.ldy + n] = f2bf(s + (a.bias ? bf2f(a.bias[n]) : 0.f));
    }
  }
}

// dx = dy W for few rows, or few columns of W: 32 MT rows (MT 1 or 2; blockIdx.y) x one block of 32 columns of dx
// per workgroup, its waves taking every 16th (MT 2: 8th) 64 rows n of W, joined through LDS in wave order.  A lane
// holds a row's block of 32 codes; the sum runs over rows, so the wave turns its 64 x 32 through LDS as bf16
// (exact) for the bf16 MFMA.  dy is rounded to bf16 on its way.  One launch, W read once per row group in four
// bits, no W in bf16 in memory.
// dy, which every workgroup reads whole, sets the time, so a wave loads whole rows of it, 128 B of eight rows an
// instruction, and takes the operands from LDS: 64 x 5120 x 5120 16 us, 22 with the operands loaded as they are used (32
// pieces of 32 B an instruction; 1599 x 7445 x 608, rows of odd length: 53 us against 149).  MT 2 with 16 waves,
// whose registers then leave room for one workgroup a CU: 22 us; MT 1 with 8: 11.0 instead of 9.9 us (32 rows).  Loads
// issued earlier, one or two pieces ahead of their use, are no faster.
constexpr int DX_PITCH = 80;              // bytes of a row of 32 bf16 in LDS: 16-byte accesses of 16 rows meet no bank twice
constexpr int DY_PITCH = 144;             // the same of a row of 64 bf16 of dy
constexpr int dx_waves(int MT) { return MT == 1 ? 16 : 8; }

template <typename T, int MT>
__global__ __launch_bounds__(64 * dx_waves(MT)) void mx_dx_rows_kernel(const T* __restrict__ dy, int64_t lddy,
                                                                   const uint8_t* __restrict__ wq,
                                                                   const uint8_t* __restrict__ ws,
                                                                   bf16* __restrict__ dx, int64_t lddx,
                                                                   int64_t rows, int N, int K, int steps) {
  constexpr int WAVES = dx_waves(MT);
  constexpr int TILE = MT * 32 * DY_PITCH > 64 * DX_PITCH ? MT * 32 * DY_PITCH : 64 * DX_PITCH;
  __shared__ __attribute__((aligned(16))) char smem[WAVES * TILE];
  const int lane = threadIdx.x & 63, blk = lane >> 5;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kb = blockIdx.x, pieces = (N + 63) / 64;
  const int64_t g = blockIdx.y;
  const int M = (int)min(rows - g * 64, (int64_t)64);
  // lane l takes row l of the piece
  const int kl = (kb & 1) * 32 + (lane & 31), kh = (kb >> 1) & 1;
  const uint8_t* w = wq + (int64_t)(kb >> 2) * PIECE + blk * 2048 + kh * 1024 + kl * 16;
  const uint8_t* sw = ws + (int64_t)(kb >> 2) * PIECE_S + kl * 4 + blk * 2 + kh;
  char* tile = smem + wid * TILE;
  const char* turned = tile + (8 * blk + ((lane >> 2) & 3)) * DX_PITCH + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
  f32x16 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = (f32x16)(0.f);
  typedef typename Loaded<T, 8>::vec raw8;
  u32x4 wv;
  uint32_t sv;
  raw8 d[MT * 4];
  // dy in runs of whole rows: lane l loads columns 8 (l % 8) of row l / 8 of every eighth row
  const T* s = dy + (g * 64 + (lane >> 3)) * lddy + (lane & 7) * 8;
  auto load = [&](int p) {
    if (p >= pieces) return;
    wv = *(const u32x4*)(w + (int64_t)p * steps * PIECE);
    sv = sw[(int64_t)p * steps * PIECE_S];
    const int have = N - p * 64 - (lane & 7) * 8;
#pragma unroll
    for (int i = 0; i < MT * 4; ++i) {
      if (i * 8 >= M) continue;
      const T* q = s + i * 8 * lddy + p * 64;
      if (i * 8 + (lane >> 3) >= M) {
      } else if (have >= 8) {
        d[i] = *(const typename Loaded<T, 8>::at*)q;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) d[i][k] = k < have ? q[k] : (T)0.f;
      }
    }
  };
  load(wid);
  for (int p = wid; p < pieces; p += WAVES) {
#pragma unroll
    for (int i = 0; i < MT * 4; ++i) {
      if (i * 8 >= M) continue;
      bf16x8 t;
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = (bf16)(float)d[i][k];
      *(bf16x8*)(tile + (i * 8 + (lane >> 3)) * DY_PITCH + (lane & 7) * 16) = t;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    bf16x8 y[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[m][e] = *(const bf16x8*)(tile + (m * 32 + (lane & 31)) * DY_PITCH + e * 32 + blk * 16);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const float scale = scale_value(sv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf16x8 t;
      const uint32_t c = wv[i];
      const auto a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0);
      const auto a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1);
      const auto a2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2);
      const auto a3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3);
      t[0] = (bf16)(a0[0] * scale), t[1] = (bf16)(a0[1] * scale), t[2] = (bf16)(a1[0] * scale);
      t[3] = (bf16)(a1[1] * scale), t[4] = (bf16)(a2[0] * scale), t[5] = (bf16)(a2[1] * scale);
      t[6] = (bf16)(a3[0] * scale), t[7] = (bf16)(a3[1] * scale);
      *(bf16x8*)(tile + lane * DX_PITCH + i * 16) = t;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bf16x8 t = cat8(lds_read_tr(turned + e * 16 * DX_PITCH), lds_read_tr(turned + (e * 16 + 4) * DX_PITCH));
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] = mfma32(t, y[m][e], acc[m]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    load(p + WAVES);
  }
  // register 4 q + c of lane l is column 8 q + 4 (l / 32) + c of row l % 32
  float* part = (float*)smem;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 v = {acc[m][4 * q], acc[m][4 * q + 1], acc[m][4 * q + 2], acc[m][4 * q + 3]};
      *(f32x4*)(part + wid * 1024 + q * 256 + lane * 4) = v;
    }
    __syncthreads();
#pragma unroll
    for (int t = threadIdx.x; t < 1024; t += 64 * WAVES) {
      const int l = (t >> 2) & 63, mm = m * 32 + (l & 31), k = kb * 32 + 8 * (t >> 8) + 4 * (l >> 5) + (t & 3);
      if (mm < M && k < K) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) s += part[i * 1024 + t];
        dx[(g * 64 + mm) * lddx + k] = f2bf(s);
      }
    }
  }
}

// The tiled product: 64 WT x 64 WT of y per workgroup, four waves of 32 WT x 32 WT each.  Every step of
// 128 columns (PIECE bytes a row piece) lands in a four-slot LDS ring by LDS-DMA, three steps ahead;
// operands are in MFMA order already, so a piece is copied as it lies and every fragment is one
// ds_read_b128 in lane order (no bank conflicts, no address arithmetic).
//   step j: wait for the own DMA of step j+1 | barrier | DMA of step j+3 into the slot of step j-1
//           | MFMAs of column half 0 beside the reads of half 1 | MFMAs of half 1 beside the reads
//           of step j+1's half 0
// RAW: step j+1 is read after the barrier that every wave passes with its part of it landed.  WAR: the
// slot of step j-1 was read for MFMAs that precede this barrier in every wave.  Past the last
// step the DMA fetches it again into a slot nobody reads, so the count is the same every step.
//
// WT 4: 32760 x 13824 x 5120 takes 1.10 ms = 4.2 PFLOP/s.  MFMAs alone on random operands run at 6.0 to 6.6 PFLOP/s (the
// clock falls to 1.5 GHz); here they are busy 57 % of 1.78 GHz.  A tile takes 65 k cycles: first loads 2.9 k, 40 steps
// of 1316 (1024 of MFMAs), image 3.7 k, stores 4.9 k, the next workgroup 1.3 k.  Two things bound it.  The operands' way
// into LDS: without the DMA it takes 0.84 ms (from a few KiB of L2 instead of HBM still 1.08, so not HBM).  And power,
// which gives fewer cycles a lower clock: 1.10 ms each, measured and dropped, were one workgroup per CU walking its
// tiles as one stream of steps, the finished tile stored during the next one's, and the 16 x 16 x 128 MFMAs (alone 13 %
// faster), at 1.90 GHz for more cycles.
// WT 2: LDS sets the time, 48 KiB a step per CU against 256 cycles of MFMAs (512 x 5120 x 4096: 12 us, of which 5 us are
// launch, first loads and stores).  Measured and dropped, no faster: an eight-slot ring, fragments read a whole
// step ahead, and two groups of waves that share K.
template <int WT>
__global__ __launch_bounds__(NT, WT == 4 ? 1 : 2) void mx_gemm_tile_kernel(MxArgs a) {
  constexpr int OPB = WT * PIECE, OPS = WT * PIECE_S, SLOT = 2 * (OPB + OPS);
  __shared__ __attribute__((aligned(16))) char smem[4 * SLOT];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wid >> 1, wm = wid & 1;
  int tm, tn;
  tile_of(blockIdx.x, (int)((a.M + 64 * WT - 1) / (64 * WT)), (a.N + 64 * WT - 1) / (64 * WT), tm, tn);
  const int steps = a.steps;

  // DMA sources: a wave moves WT KiB of each operand and (WT 4: of both, WT 2: of one) 256 B of scales
  // a step.  Row pieces past the matrix are clamped to its last (their results are not stored).
  const int gn = (a.N + 63) / 64;
  const int64_t gm = (a.M + 63) / 64;
  const int own = WT == 4 ? wid : wid >> 1;             // row piece of the tile
  const int part = WT == 4 ? 0 : (wid & 1) * 2048;
  const int64_t pn = min(tn * WT + own, gn - 1), pm = min((int64_t)tm * WT + own, gm - 1);
  const uint32_t bytes = (uint32_t)steps * PIECE;
  const i32x4 srd_w = make_srd(a.wq + pn * steps * PIECE + part, bytes - part);
  const i32x4 srd_x = make_srd(a.xq + pm * steps * PIECE + part, bytes - part);
  const int64_t sn = min(tn * WT + (WT == 4 ? wid : wid & 1), gn - 1);
  const int64_t sm = min((int64_t)tm * WT + (WT == 4 ? wid : wid & 1), gm - 1);
  const i32x4 srd_sw = make_srd(a.ws + sn * steps * PIECE_S, (uint32_t)steps * PIECE_S);
  const i32x4 srd_sx = make_srd(a.xs + sm * steps * PIECE_S, (uint32_t)steps * PIECE_S);
  const uint32_t lds0 = lds_addr(smem);
  unsigned keep = 0;
  // DMA p of the step's DMAS
  constexpr int DMAS = WT == 4 ? 10 : 5;
  auto dma = [&](int p, int j) {
    const uint32_t at = lds0 + (uint32_t)(j & 3) * SLOT, k = (uint32_t)min(j, steps - 1);
    if (p < 2 * WT) {
      const int op = p >= WT, i = p - op * WT;
      if (i == 0) m0_set(at + op * OPB + wid * (WT * 1024), keep);
      dma16_buf_m0(op ? srd_x : srd_w, lane * 16, k * PIECE, i);
      if (i == WT - 1) m0_restore(keep);
    } else {
      const bool op = WT == 4 ? p == 2 * WT + 1 : wid >= 2;
      const int i = WT == 4 ? wid : wid & 1;
      m0_set(at + 2 * OPB + (op ? OPS : 0) + i * PIECE_S, keep);
      dma4_step(op ? srd_sx : srd_sw, lane * 4, k * PIECE_S);
      m0_restore(keep);
    }
  };

  f32x16 acc[WT][WT];
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < WT; ++j) acc[i][j] = (f32x16)(0.f);
  u32x4 f[2][2][WT];                     // [column half][W, x][tile]
  uint32_t sc[2][2][WT / 2];             // [step parity][W, x][row piece]
  // fragment r (< 2 WT) of half h, step j: the wave's row pieces start at wn (wm) * WT / 2
  auto read = [&](int r, int h, int j) {
    const int op = r >= WT, i = r - op * WT;
    const char* st = smem + (j & 3) * SLOT + op * OPB + (op ? wm : wn) * (WT / 2) * PIECE;
    f[h][op][i] = *(const u32x4*)(st + (i >> 1) * PIECE + ((i & 1) * 2 + h) * 1024 + lane * 16);
  };
  auto read_scales = [&](int par, int j) {
#pragma unroll
    for (int op = 0; op < 2; ++op)
#pragma unroll
      for (int i = 0; i < WT / 2; ++i)
        sc[par][op][i] = *(const uint32_t*)(smem + (j & 3) * SLOT + 2 * OPB + op * OPS +
                                            ((op ? wm : wn) * (WT / 2) + i) * PIECE_S + lane * 4);
  };
  // MFMA c of a half: tile pair (c / 4), then the four of its 2 x 2 tiles
  auto product = [&](auto half, int par, int c) {
    constexpr int H = half();
    const int ii = c / 4 / (WT / 2), jj = c / 4 % (WT / 2), q = c & 3;
    const uint32_t sw = sc[par][0][ii], sx = sc[par][1][jj];
    f32x16& d = acc[2 * ii + (q >> 1)][2 * jj + (q & 1)];
    const u32x4 w = f[H][0][2 * ii + (q >> 1)], x = f[H][1][2 * jj + (q & 1)];
    if (q == 0) d = mfma4<H, H>(w, x, d, sw, sx);
    else if (q == 1) d = mfma4<H, 2 + H>(w, x, d, sw, sx);
    else if (q == 2) d = mfma4<2 + H, H>(w, x, d, sw, sx);
    else d = mfma4<2 + H, 2 + H>(w, x, d, sw, sx);
  };
  auto step = [&](auto parity, int j) {
    constexpr int P = parity();
    if constexpr (DMAS == 10) asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(5)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int c = 0; c < WT * WT; ++c) {
      product(std::integral_constant<int, 0>(), P, c);
      if (c < 2 * WT) read(c, 1, j);
      if (c < DMAS) dma(c, j + 3);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int c = DMAS < WT * WT ? DMAS : WT * WT; c < DMAS; ++c) dma(c, j + 3);
    read_scales(1 - P, j + 1);
#pragma unroll
    for (int c = 0; c < WT * WT; ++c) {
      product(std::integral_constant<int, 1>(), P, c);
      if (c < 2 * WT) read(c, 0, j + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int j = 0; j < 3; ++j)
#pragma unroll
    for (int p = 0; p < DMAS; ++p) dma(p, j);
  if constexpr (DMAS == 10) asm volatile("s_waitcnt vmcnt(20)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int r = 0; r < 2 * WT; ++r) read(r, 0, 0);
  read_scales(0, 0);
  int j = 0;
  for (; j + 1 < steps; j += 2) {
    step(std::integral_constant<int, 0>(), j);
    step(std::integral_constant<int, 1>(), j + 1);
  }
  if (j < steps) step(std::integral_constant<int, 0>(), j);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  const int n0 = tn * 64 * WT + wn * 32 * WT;
  const int64_t m0 = (int64_t)tm * 64 * WT + wm * 32 * WT;
  // The tile leaves through a wave-private LDS image (16 B of padding a row), so that a store instruction writes
  // whole lines; in the MFMA layout it would write 64 pieces of 8 B (32760 x 13824 x 5120: 1.77 ms so, 1.16 ms
  // through the image).  Non-temporal, past the operands in L2 (1.20 ms without).  Rows need not be aligned.
  constexpr int ROW = 64 * WT + 16, LPR = 4 * WT, RPI = 64 / LPR;
  static_assert(4 * WT * 32 * ROW <= 4 * SLOT, "the images reuse the ring");
  bf16x4 b[WT][4];
  if (a.bias && (tn + 1) * 64 * WT <= a.N) {
#pragma unroll
    for (int i = 0; i < WT * 4; ++i)
      b[i >> 2][i & 3] = *(const typename Loaded<bf16, 4>::at*)(a.bias + n0 + i * 8 + 4 * (lane >> 5));
  } else {
#pragma unroll
    for (int i = 0; i < WT * 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = n0 + i * 8 + 4 * (lane >> 5) + k;
        b[i >> 2][i & 3][k] = a.bias && n < a.N ? a.bias[n] : (bf16)0.f;
      }
  }
  __builtin_amdgcn_s_barrier();            // every wave's DMA has landed and its fragments are read
  asm volatile("" ::: "memory");
  char* img = smem + wid * (WT * 32 * ROW);
#pragma unroll
  for (int jj = 0; jj < WT; ++jj)
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        bf16x4 o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = f2bf(acc[i][jj][4 * r + k] + bf2f(b[i][r][k]));
        *(bf16x4*)(img + (jj * 32 + (lane & 31)) * ROW + (i * 32 + 8 * r + 4 * (lane >> 5)) * 2) = o;
      }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const int n = n0 + (lane % LPR) * 8;
  bf16* const y0 = a.y + (m0 + lane / LPR) * a.ldy + n;
  const bool inside = (tn + 1) * 64 * WT <= a.N && (int64_t)(tm + 1) * 64 * WT <= a.M;
#pragma unroll
  for (int t0 = 0; t0 < WT * 32 / RPI; t0 += 8) {
    bf16x8 o[8];
#pragma unroll
    for (int t = 0; t < 8; ++t)
      o[t] = *(const bf16x8*)(img + ((t0 + t) * RPI + lane / LPR) * ROW + (lane % LPR) * 16);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      bf16* p = y0 + (int64_t)(t0 + t) * RPI * a.ldy;
      if (inside || (m0 + (t0 + t) * RPI + lane / LPR < a.M && n + 8 <= a.N)) {
        __builtin_nontemporal_store(o[t], (typename Loaded<bf16, 8>::at*)p);
      } else if (m0 + (t0 + t) * RPI + lane / LPR < a.M) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (n + k < a.N) p[k] = o[t][k];
      }
    }
  }
}

// Which kernel, by measured kernel times in us (rows / 128 tile, K 5120 where none is named):
//   mx_rows_kernel while its workgroups come in about one round of the chip (at most 256; up to 384 where K is
//   long, where a tile's own loop is what takes time; for 32 rows, whose workgroups are half the work, 512):
//     32 x 5120  4.5 / 11.8    32 x 13824  10.7 / 13.2    64 x 5120 6.0 / 11.8   64 x 10240 11.0 / 12.3   64 x 13824
//     13.9 / 13.5    192 x 4096 10.5 / 12.0 (K 1280: 7.1 / 6.1)    256 x 1280 6.1 / 11.1    512 x 1280 10.3 / 11.7
//     128 x 8192 (K 4096) 15.0 / 10.2    300 x 100 (K 14000) 9.4 / 25.8    768 x 1024 (K 13824) 21.0 / 27.5
//     16 x 65536 (K 4096) 36 / 24
//   else the tile whose rounds of the chip take less: 256 tiles of 256 at a time take 8.5 + 0.82 us a step of K, 512 of
//   128, two a CU, whose loads and stores overlap, 2.5 + 0.51 (256 / 128 tile; tiles of 256):
//     4096 x 4096 (256) 43 / 47 (K 1280: 18.3 / 17.4)    4352 x 5120 (340) 74 / 68    2048 x 13824 (432) 81 / 83    6000 x 5120
//     (480) 84.5 / 93    7258 x 4808 (551) 132 / 125 (K 1280: 58 / 48)    8190 x 5120 (640) 120 / 122    6400 x 8192 (800)
//     166 / 169 (K 640: 47 / 35)    8960 x 7680 (1050) 210 / 221    16000 x 5120 (1260) 213 / 234
//     12359 x 2272, K 1760 (441) 47 / 39    17996 x 9984, K 1792 (2769) 240 / 248
bool by_rows(int64_t M, int64_t N, int steps) {
  const int64_t n = ((M + 63) / 64) * ((N + 31) / 32);
  return n <= 256 || (n <= 384 && steps >= 20) || (M <= 32 && n <= 512);
}

void launch_product(const MxArgs& a, hipStream_t st) {
  const int64_t t256 = ((a.M + 255) / 256) * ((a.N + 255) / 256), t128 = ((a.M + 127) / 128) * ((a.N + 127) / 128);
  const int64_t us256 = ((t256 + 255) / 256) * (850 + 82 * a.steps), us128 = ((t128 + 511) / 512) * (250 + 51 * a.steps);
  const dim3 cols((unsigned)((a.N + 31) / 32), (unsigned)((a.M + 63) / 64));
  if (by_rows(a.M, a.N, a.steps)) {
    if (a.M <= 32)
      hipLaunchKernelGGL((mx_rows_kernel<bf16, 1, false>), cols, dim3(64 * ROWS_WAVES), 0, st, a, nullptr, 0, 0);
    else
      hipLaunchKernelGGL((mx_rows_kernel<bf16, 2, false>), cols, dim3(64 * ROWS_WAVES), 0, st, a, nullptr, 0, 0);
  } else if (us256 < us128) {
    hipLaunchKernelGGL(mx_gemm_tile_kernel<4>, dim3((unsigned)t256), dim3(NT), 0, st, a);
  } else {
    hipLaunchKernelGGL(mx_gemm_tile_kernel<2>, dim3((unsigned)t128), dim3(NT), 0, st, a);
  }
}

// One launch for both: every workgroup quantises all of x, so only while that is a block a thread.  Kernel times in us
// against two launches (rows x columns of y x K): 1 x 5120 x 5120 4.4 / 7.7, 6 x 5120 x 5120 5.5 / 7.7, 1 x 13824 x 5120
// 10.8 / 13.4, 1 x 30000 x 4096 18.2 / 17.5.  The columns are not in the rule, though each workgroup of 32 of them
// quantises x again: 8 x 13824 x 4096 15.0 / 13.3, 8 x 65536 x 4096 55 / 27.
bool fused(int64_t M, int64_t K) { return M <= 32 && M * ((K + 31) / 32) <= ROWS_FUSED; }

// dx in one launch while its workgroups are few: kernel times in us against W read back to bf16 and multiplied by the
// tiled bf16 product (M x N x K): 1 x 5120 x 5120 7.9 / 85, 64 x 5120 x 5120 16 / 86, 128 (320 workgroups) 31 / 87, 256
// (640) 48 / 87; 2 x 13312 x 96 15 / 184; 512 x 1280 x 1280 (320) 12.2 / 26.3; 2048 x 640 x 640 (640) 13.5 / 16.8;
// 512 x 13824 x 4000 (1000) 163 / 215; 512 x 640 x 5120 (1280) 21.8 / 19.1.  A single group of 64 rows reads W once either
// way, here in four bits, and stays here whatever its width: 64 x 14000 x 13824 83 / 335, 32 x 8192 x 30000 54 / 304.
constexpr int DX_DIRECT = 1024;

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
  prfl_prof::begin(KID_GEMM, st);
  launch_product(a, st);
  prfl_prof::set_work(2.0 * M * N * K);
  prfl_prof::end(KID_GEMM, st);
  PRFL_LAUNCH_CHECK();
  return 0;
}

extern "C" int64_t prfl_linear_mxfp4_ws_bytes(int64_t M, int64_t K) {
  if (M <= 0 || too_large(M, K) || fused(M, K)) return 0;
  return ((M + 63) / 64) * ((K + 127) / 128) * (PIECE + PIECE_S);
}

extern "C" int prfl_linear_mxfp4(const void* x, int x_type, int64_t ldx, const void* wq, const void* ws,
                                 const void* bias, void* y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                                 void* work, int64_t work_bytes, void* stream) {
  const int64_t need = prfl_linear_mxfp4_ws_bytes(M, K);
  if (x_type < 0 || x_type > 2 || (M > 1 && ldx < 0) || work_bytes < need || (need && !work))
    return (int)hipErrorInvalidValue;
  if (need || M <= 0) {
    uint8_t* xs = (uint8_t*)work + need / (PIECE + PIECE_S) * PIECE;
    if (need)
      if (int rc = prfl_quant_mxfp4(x, x_type, ldx, M, K, work, xs, stream)) return rc;
    return prfl_gemm_mxfp4(work, xs, wq, ws, bias, y, ldy, M, N, K, stream);
  }
  if (too_large(M, K) || too_large(N, K) || N < 1 || N > (1 << 24) || (M > 1 && ldy < N) || !x || !wq || !ws || !y ||
      ((uintptr_t)wq & 15) || ((uintptr_t)ws & 3))
    return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  MxArgs a{(const uint8_t*)wq, (const uint8_t*)ws, nullptr, nullptr, (const bf16*)bias, (bf16*)y, ldy, M,
           (int)N, (int)((K + 127) / 128)};
  const dim3 cols((unsigned)((N + 31) / 32));
  prfl_prof::begin(KID_GEMM, st);
  if (x_type == 0)
    hipLaunchKernelGGL((mx_rows_kernel<float, 1, true>), cols, dim3(64 * ROWS_WAVES), 0, st, a, (const float*)x, ldx,
                       (int)K);
  else if (x_type == 1)
    hipLaunchKernelGGL((mx_rows_kernel<bf16, 1, true>), cols, dim3(64 * ROWS_WAVES), 0, st, a, (const bf16*)x, ldx,
                       (int)K);
  else
    hipLaunchKernelGGL((mx_rows_kernel<_Float16, 1, true>), cols, dim3(64 * ROWS_WAVES), 0, st, a, (const _Float16*)x,
                       ldx, (int)K);
  prfl_prof::set_work(2.0 * M * N * K);
  prfl_prof::end(KID_GEMM, st);
  PRFL_LAUNCH_CHECK();
  return 0;
}

extern "C" int prfl_linear_mxfp4_dx_direct(int64_t M, int64_t N, int64_t K) {
  return M > 0 && N > 0 && K > 0 && (M <= 64 || ((M + 63) / 64) * ((K + 31) / 32) <= DX_DIRECT);
}

extern "C" int prfl_linear_mxfp4_dx(const void* dy, int y_type, int64_t lddy, const void* wq, const void* ws,
                                    void* dx, int64_t lddx, int64_t M, int64_t N, int64_t K, void* stream) {
  if (too_large(M, K) || too_large(N, K) || N < 1 || N > (1 << 24) || y_type < 0 || y_type > 2 ||
      (M > 1 && (lddy < 0 || lddx < K)) || (M + 63) / 64 > 65535)
    return (int)hipErrorInvalidValue;
  if (M == 0) return 0;
  if (!dy || !wq || !ws || !dx || ((uintptr_t)wq & 15)) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)((K + 31) / 32), (unsigned)((M + 63) / 64));
  const int steps = (int)((K + 127) / 128);
  auto run = [&](auto* p) {
    if (M <= 32)
      hipLaunchKernelGGL((mx_dx_rows_kernel<std::remove_const_t<std::remove_pointer_t<decltype(p)>>, 1>), grid,
                         dim3(64 * dx_waves(1)), 0, st, p, lddy, (const uint8_t*)wq, (const uint8_t*)ws, (bf16*)dx,
                         lddx, M, (int)N, (int)K, steps);
    else
      hipLaunchKernelGGL((mx_dx_rows_kernel<std::remove_const_t<std::remove_pointer_t<decltype(p)>>, 2>), grid,
                         dim3(64 * dx_waves(2)), 0, st, p, lddy, (const uint8_t*)wq, (const uint8_t*)ws, (bf16*)dx,
                         lddx, M, (int)N, (int)K, steps);
  };
  prfl_prof::begin(KID_GEMM, st);
  if (y_type == 0) run((const float*)dy);
  else if (y_type == 1) run((const bf16*)dy);
  else run((const _Float16*)dy);
  prfl_prof::set_work(2.0 * M * N * K);
  prfl_prof::end(KID_GEMM, st);
  PRFL_LAUNCH_CHECK();
  return 0;
}
