// int8_linear.hip — rows quantised to int8 with one scale per token, and their
// product with int8 weights of one scale per output channel.
//
// Mathematics.  y[m, n] = xs[m] ws[n] sum_k xc[m, k] wc[n, k] + b[n], xs = max|x| /
// 127, xc = rn(127 x / max|x|) (ties to even, the rounding of the exact quotient; of
// a row with gamma that of fp32 products, so that a code next to a border may be its
// neighbour).  Of an RMS-normalised row x r gamma, r = 1 / sqrt(mean x^2 + eps), the
// codes do not depend on r: they are those of x gamma, and r multiplies the scale.  So one
// pass over the row gives maximum and sum of squares together, and nothing is rounded
// between norm and code.  The sums are exact in 32-bit integers: 128^2 k < 2^31
// for k < 131072.  What follows is fp32, rounded to bf16 once.
//
// Rows are held in registers between the pass for the maximum and the codes: 2 bytes
// read and 1 written per value, bound by HBM for many rows (8191 x 8192 with a norm
// 41-45 us, 4.5-4.9 TB/s; a large copy moves 4.97), by launch and two dependent loads
// for few (64 x 4096: 4.0 us).  The next row is under way while one is reduced.
//
// Products.  The larger a tile, the less is copied to LDS and read from it per
// product (a CU copies up to 140 KB/us of what lies in L2); but there are 256 CUs to
// fill.  Hence forms of many tile sizes, chosen by measured costs (kForms), all with
// v_mfma_i32_32x32x32_i8 but the one that streams the weights for 16 rows or fewer.
// Two times: weights from memory (a model's, more than the 256 MB that the memory-side
// cache holds), in brackets weights found there:
//   256 x 256, waves that take turns: bound by power.  8191 x 8192 x 10240: 565-595 us by card,
//     2.3-2.4 POP/s, the matrix units busy 70 % of the cycles at a clock that falls to 1.7
//     GHz; the library's product of two 8192^3 int8 matrices reaches 2.15.
//   192, 160, 128 and 64 x 128, 64 x 64, ring of tiles read and copied ahead: 517 x 2880 x
//     5120 17.3 us (14.2-15.3), bound by the 200 tiles' 23 steps and the start.
//   32 x 64, 32 x 32, four groups of waves with a quarter of k each: latency of the copies.
//     64 x 4096 x 6144 11.3 us (8.1), 2.2 TB/s of weights.
//   16 rows or fewer, operands straight to registers: 4 x 2048 x 2048 3.9 us (3.4:
//     launch and one load); 16 x 4096 x 4096 7.1 us (6.2).
// LDS tiles hold rows of 128 (256 x 256: 64, 64 x 64: 256) bytes of k in 16-byte chunks, exchanged
// within a row so that the 16 rows that a fragment read touches at once lie in all
// banks (conflicts: 3 % of the LDS cycles).
#include <algorithm>
#include <atomic>

#include "attn_tile.h"

namespace mia {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) uint16_t lds_u16_t;

// ---------------------------------------------------------------------------
// rows to int8
// ---------------------------------------------------------------------------
MIA_DEV float add_bf16(float a, float b) { return bf16lo(pack2_bf16(a + b, 0.f)); }

// The squares of a row have left fp32 where their sum is an infinity (values from
// 2^60 on or so), or so small that what it lost counts: an eps from 2^-75 on is
// 2^25 times it and more.
MIA_DEV bool squares_left(float ss, const mia_quant_rows_args &a) {
  return !(ss <= 3.402823466e38f && ss >= (a.eps < 0x1p-75f ? 0x1p-100f : 0.f));
}

// 1 / rms, times f, of squares of the values times f.
MIA_DEV float inverse_rms(float ss, float f, const mia_quant_rows_args &a) {
  const float n = (float)(a.dim_actual > 0 ? a.dim_actual : a.dim);
  return 1.0f / sqrtf(ss / n + a.eps * f * f);
}

// The row's scale: fl32(amax / 127), of the normalised row; -amax where its squares
// have left fp32 (`left`).
MIA_DEV float row_scale(uint32_t mag, float ss, bool left, const mia_quant_rows_args &a) {
  if (mag >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  float amax = __uint_as_float(mag);
  if (a.norm) {
    if (mag == 0) return 0.f;  // (without an eps it would be 0 times an infinity)
    if (left) return -amax;
    amax *= inverse_rms(ss, 1.0f, a);
  }
  return amax / 127.0f;
}

MIA_DEV float gamma_at(const mia_quant_rows_args &a, int c) {
  if (a.gamma_bf16) return bf16_bits_to_f32(((const uint16_t *)a.gamma)[c]);
  return ((const float *)a.gamma)[c];
}

// Channel c of the row at `at`, with its residual adds.
MIA_DEV float row_value(const mia_quant_rows_args &a, int64_t at, int c) {
  float x = bf16_bits_to_f32(((const uint16_t *)a.x)[at + c]);
  if (a.add0) x = add_bf16(x, bf16_bits_to_f32(((const uint16_t *)a.add0)[at + c]));
  if (a.add1) x = add_bf16(x, bf16_bits_to_f32(((const uint16_t *)a.add1)[at + c]));
  return x;
}

// The scale of a row whose squares have left fp32, -amax so far, by a second read:
// squares of the values times 2^-80 (at most 2^96 each, 2^-32 of a sum that was an
// infinity) or 2^80 (2^-106 to 2^60).  The row's LANES threads call it; sums: their
// waves'.  No part of the rows' own loop, which it would cost registers and 2 to 14 %.
template <int LANES>
MIA_DEV void scale_again(const mia_quant_rows_args &a, int64_t row, int tid, float2 *sums) {
  float lo = 0.f, hi = 0.f;
  int c = tid;
  asm volatile("" : "+v"(c));  // (addresses are formed here, not before the rows' loop)
#pragma nounroll
  for (; c < a.dim; c += LANES) {
    const float x = row_value(a, row * a.x_stride, c);
    lo = fmaf(x * 0x1p-80f, x * 0x1p-80f, lo);
    hi = fmaf(x * 0x1p80f, x * 0x1p80f, hi);
  }
#pragma nounroll
  for (int o = 1; o < 64; o <<= 1) {
    lo += __shfl_xor(lo, o, 64);
    hi += __shfl_xor(hi, o, 64);
  }
  if constexpr (LANES == 256) {
    __syncthreads();  // (those of the row before have been read)
    if ((tid & 63) == 0) sums[tid >> 6] = make_float2(lo, hi);
    __syncthreads();
    lo = (sums[0].x + sums[1].x) + (sums[2].x + sums[3].x);
    hi = (sums[0].y + sums[1].y) + (sums[2].y + sums[3].y);
  }
  if (tid != 0) return;
  const float amax = -a.scales[row];
  if (!(amax > 0.f)) return;  // (another row's squares have)
  // (small values' sum is below 2^60 of them, large ones' an infinity or beyond)
  const bool small = hi < 0x1p100f;
  const float f = small ? 0x1p80f : 0x1p-80f;
  a.scales[row] = amax * f * inverse_rms(small ? hi : lo, f, a) / 127.0f;
}

// LANES threads per row, NV vectors of 8 channels each, held in registers.  With
// NORM a workgroup takes rows row0, row0 + stride, ...: gamma, twice the bytes of
// a row where it is fp32, is loaded once for all of them.
template <int LANES, int NV, bool NORM>
__global__ __launch_bounds__(256) void quant_rows_kernel(mia_quant_rows_args a) {
  constexpr int RPB = 256 / LANES;
  __shared__ float2 red[2][4];
  __shared__ float2 sums[4];
  const int tid = threadIdx.x % LANES;
  bool left = false;  // has a row to be scaled again?
  f32x4_t gamma[NORM ? NV : 1][2];
  if (NORM) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * LANES + tid) * 8;
      gamma[v][0] = gamma[v][1] = f32x4_t{1.f, 1.f, 1.f, 1.f};
      if (c >= a.dim || !a.gamma) continue;
      if (a.gamma_bf16) {
        const u32x4_t g = *reinterpret_cast<const u32x4_t *>((const uint16_t *)a.gamma + c);
        gamma[v][0] = f32x4_t{bf16lo(g[0]), bf16hi(g[0]), bf16lo(g[1]), bf16hi(g[1])};
        gamma[v][1] = f32x4_t{bf16lo(g[2]), bf16hi(g[2]), bf16lo(g[3]), bf16hi(g[3])};
      } else {
        gamma[v][0] = *reinterpret_cast<const f32x4_t *>((const float *)a.gamma + c);
        gamma[v][1] = *reinterpret_cast<const f32x4_t *>((const float *)a.gamma + c + 4);
      }
    }
  }
  const int64_t stride = (int64_t)gridDim.x * RPB;
  const int own = LANES == 256 ? 0 : threadIdx.x / LANES;  // (0: a row of all threads is uniform)
  int64_t row = (int64_t)blockIdx.x * RPB + own;
  u32x4_t raw[NV];
  auto load = [&](int64_t r) {
    const int64_t at = (r < a.rows ? r : 0) * a.x_stride;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * LANES + tid) * 8;
      raw[v] = u32x4_t{0u, 0u, 0u, 0u};
      if (c < a.dim) raw[v] = *reinterpret_cast<const u32x4_t *>((const uint16_t *)a.x + at + c);
    }
  };
  load(row);
  // (every thread of a workgroup takes as many turns)
  for (int64_t first = (int64_t)blockIdx.x * RPB, turn = 0; first < a.rows;
       first += stride, row += stride, ++turn) {
    const bool live = row < a.rows;
    float x[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[v][2 * i] = bf16lo(raw[v][i]);
        x[v][2 * i + 1] = bf16hi(raw[v][i]);
      }
    if (first + stride < a.rows) load(row + stride);
    auto add = [&](const void *t) {
      if (!t) return;
      const int64_t at = (live ? row : 0) * a.x_stride;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * LANES + tid) * 8;
        if (c >= a.dim) continue;
        const u32x4_t w = *reinterpret_cast<const u32x4_t *>((const uint16_t *)t + at + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[v][2 * i] = add_bf16(x[v][2 * i], bf16lo(w[i]));
          x[v][2 * i + 1] = add_bf16(x[v][2 * i + 1], bf16hi(w[i]));
        }
      }
    };
    add(a.add0);
    add(a.add1);
    float ss = 0.f;
    if constexpr (NORM) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss = fmaf(x[v][i], x[v][i], ss);
          x[v][i] *= gamma[v][i >> 2][i & 3];
        }
    }
    // magnitudes as integers: an infinity or NaN is the largest
    uint32_t mag = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) mag = max(mag, __float_as_uint(x[v][i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      mag = max(mag, (uint32_t)__shfl_xor((int)mag, o, 64));
      if (NORM) ss += __shfl_xor(ss, o, 64);
    }
    if constexpr (LANES == 256) {
      float2 *const rd = red[turn & 1];
      if ((threadIdx.x & 63) == 0) rd[threadIdx.x >> 6] = make_float2(__uint_as_float(mag), ss);
      __syncthreads();
      mag = max(max(__float_as_uint(rd[0].x), __float_as_uint(rd[1].x)),
                max(__float_as_uint(rd[2].x), __float_as_uint(rd[3].x)));
      ss = (rd[0].y + rd[1].y) + (rd[2].y + rd[3].y);
    }
    if (!live) continue;
    RowCodes<127> rs;
    rs.set(mag);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * LANES + tid) * 8;
      if (c >= a.dim) continue;
      u32x2_t w = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i >> 2] |= rs.int8(x[v][i]) << (8 * (i & 3));
      *reinterpret_cast<u32x2_t *>((uint8_t *)a.codes + row * a.codes_stride + c) = w;
    }
    const bool again = NORM && mag - 1u < 0x7f7fffffu && squares_left(ss, a);
    if (tid == 0) a.scales[row] = row_scale(mag, ss, again, a);
    left |= again;
  }
  if (NORM && left)  // (the same for a row's threads)
    for (row = (int64_t)blockIdx.x * RPB + own; row < a.rows; row += stride)
      scale_again<LANES>(a, row, tid, sums);
}

// Any width, alignment and length: a workgroup takes a row at a time, read twice.
__global__ __launch_bounds__(256) void quant_rows_any_kernel(mia_quant_rows_args a) {
  __shared__ float2 red[2][4];
  __shared__ float2 sums[4];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const int64_t at = row * a.x_stride;
    float ss = 0.f;
    auto value = [&](int c, bool sum) {
      const float x = row_value(a, at, c);
      if (sum) ss = fmaf(x, x, ss);
      return a.norm && a.gamma ? x * gamma_at(a, c) : x;
    };
    uint32_t mag = 0;
    for (int c = threadIdx.x; c < a.dim; c += 256)
      mag = max(mag, __float_as_uint(value(c, true)) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      mag = max(mag, (uint32_t)__shfl_xor((int)mag, o, 64));
      ss += __shfl_xor(ss, o, 64);
    }
    float2 *const rd = red[turn];
    if ((threadIdx.x & 63) == 0) rd[threadIdx.x >> 6] = make_float2(__uint_as_float(mag), ss);
    __syncthreads();
    mag = max(max(__float_as_uint(rd[0].x), __float_as_uint(rd[1].x)),
              max(__float_as_uint(rd[2].x), __float_as_uint(rd[3].x)));
    ss = (rd[0].y + rd[1].y) + (rd[2].y + rd[3].y);
    RowCodes<127> rs;
    rs.set(mag);
    for (int c = threadIdx.x; c < a.dim; c += 256)
      ((uint8_t *)a.codes)[row * a.codes_stride + c] = (uint8_t)rs.int8(value(c, false));
    const bool again = a.norm && squares_left(ss, a);
    if (threadIdx.x == 0) a.scales[row] = row_scale(mag, ss, again, a);
    if (again) scale_again<256>(a, row, threadIdx.x, sums);
  }
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------
struct GemmParams {
  const uint8_t *x, *w;
  int64_t x_ld, w_ld;  // bytes
  const float *xs, *ws;
  const void *bias;
  int bias_bf16;
  uint16_t *out;
  int64_t out_ld;
  int m, n, k;
  int mt, nt;  // tiles
  int vec;     // rows of out take 16-byte stores
};

MIA_DEV float bias_at(const GemmParams &p, int n) {
  if (!p.bias) return 0.f;
  return p.bias_bf16 ? bf16_bits_to_f32(((const uint16_t *)p.bias)[n]) : ((const float *)p.bias)[n];
}

// The workgroup's tile (column, row).  Each XCD (workgroups go round robin over
// 8) takes a contiguous run of the tiles, in groups of 8 row tiles, so that its
// L2 holds what they share.
MIA_DEV int2 tile_of(const GemmParams &p) {
  const int total = p.mt * p.nt;
  const int full = total / 8, rem = total % 8, xcd = blockIdx.x % 8;
  const int id = xcd * full + min(xcd, rem) + blockIdx.x / 8;
  const int gsz = 8 * p.nt;
  const int g = id / gsz, first = g * 8, rows = min(p.mt - first, 8);
  const int r = id - g * gsz;
  return make_int2(r / rows, first + r % rows);
}

// out = acc xs ws + bias of the workgroup's tile, rounded to bf16 through LDS so
// that rows are stored whole.  acc: TN x TM products of 32 x 32 of wave (wn, wm),
// lane: row (token) lane % 32, channels 8 g + 4 (lane / 32) ...  Every thread
// calls it, those with `has` hold sums.  LDS is free.
template <int TN, int TM, int BN, int THREADS>
MIA_DEV void store_tile(const GemmParams &p, lds_u8_t *all, const i32x16_t (&acc)[TN][TM], int n0,
                        int m0, int wn, int wm, int wave, bool has) {
  const int tid = threadIdx.x, lane = tid & 63, rl = lane & 31, half = lane >> 5;
  lds_f32_t *const wsl = (lds_f32_t *)all;  // [BN] scales, [BN] bias
  for (int i = tid; i < BN; i += THREADS) {
    const int n = min(n0 + i, p.n - 1);
    wsl[i] = p.ws[n];
    wsl[BN + i] = bias_at(p, n);
  }
  __syncthreads();
  if (!has) return;
  constexpr int ROWB = TN * 64 + 16;
  lds_u8_t *const stage = all + BN * 8 + wave * 32 * ROWB;
  const int nw = wn * TN * 32, mw = m0 + wm * TM * 32;
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const float xs = p.xs[min(mw + j * 32 + rl, p.m - 1)];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = i * 32 + g * 8 + half * 4;
        const f32x4_t s4 = *(const lds_f32x4_t *)(wsl + nw + c);
        const f32x4_t b4 = *(const lds_f32x4_t *)(wsl + BN + nw + c);
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf((float)acc[i][j][g * 4 + e] * xs, s4[e], b4[e]);
        *(lds_u32x2_t *)(stage + rl * ROWB + c * 2) =
            u32x2_t{pack2_bf16(y[0], y[1]), pack2_bf16(y[2], y[3])};
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    if (p.vec) {
      constexpr int CPR = TN * 4;  // 16-byte chunks of a row
#pragma unroll
      for (int q = 0; q < 32 * CPR / 64; ++q) {
        const int r = (q * 64 + lane) / CPR, c = (q * 64 + lane) % CPR;
        const int m = mw + j * 32 + r, n = n0 + nw + c * 8;
        const u32x4_t v = *(const lds_u32x4_t *)(stage + r * ROWB + c * 16);
        if (m < p.m && n < p.n)
          *reinterpret_cast<u32x4_t *>(p.out + (int64_t)m * p.out_ld + n) = v;
      }
    } else {
      for (int q = 0; q < 32 * TN * 32 / 64; ++q) {
        const int r = (q * 64 + lane) / (TN * 32), c = (q * 64 + lane) % (TN * 32);
        const int m = mw + j * 32 + r, n = n0 + nw + c;
        const uint16_t v = *(const lds_u16_t *)(stage + r * ROWB + c * 2);
        if (m < p.m && n < p.n) p.out[(int64_t)m * p.out_ld + n] = v;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}

// The sums of G groups of WAVES waves meet in the first group's registers, through
// LDS, which is free; at: the lane's place in its group.  Every thread calls it.
template <int G, int WAVES, int TN, int TM>
MIA_DEV void join_sums(lds_u8_t *all, i32x16_t (&acc)[TN][TM], int group, int at) {
  if constexpr (G > 1) {
    typedef __attribute__((address_space(3))) i32x4_t lds_i32x4_t;
    lds_i32x4_t *const sums = (lds_i32x4_t *)all + at;
    constexpr int PER = TN * TM * 4;
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            sums[((group - 1) * PER + (i * TM + j) * 4 + g) * WAVES * 64] =
                i32x4_t{acc[i][j][g * 4], acc[i][j][g * 4 + 1], acc[i][j][g * 4 + 2],
                        acc[i][j][g * 4 + 3]};
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int k = 1; k < G; ++k)
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const i32x4_t v = sums[((k - 1) * PER + (i * TM + j) * 4 + g) * WAVES * 64];
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][g * 4 + e] += v[e];
            }
    }
    __syncthreads();
  }
}

// LDS that join_sums needs
constexpr int join_bytes(int g, int waves, int products) {
  return (g - 1) * waves * 64 * products * 16 * 4;
}

constexpr int kBK = 128;  // bytes of k per tile

// WN x WM waves, each TN x TM products of 32 x 32, KS such groups with a share
// of k and a ring of tiles each.
template <int WN, int WM, int TN, int TM, int STAGES, int KS>
__global__ __launch_bounds__(WN *WM *KS * 64) void gemm_kernel(GemmParams p) {
  constexpr int WAVES = WN * WM;  // of a group
  constexpr int THREADS = WAVES * KS * 64;
  constexpr int BN = WN * TN * 32, BM = WM * TM * 32;
  constexpr int NC = BN / 8 / WAVES, MC = BM / 8 / WAVES;  // copies per wave and tile
  static_assert(BN % (8 * WAVES) == 0 && BM % (8 * WAVES) == 0, "whole copies");
  constexpr int STAGE = (BN + BM) * kBK;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x;
  const int group = KS == 1 ? 0 : readfirstlane(tid / (WAVES * 64));
  const int wave = readfirstlane(tid >> 6) - group * WAVES;
  const int lane = tid & 63;
  lds_u8_t *const all = (lds_u8_t *)smem;
  lds_u8_t *const lds = all + group * STAGES * STAGE;  // the group's ring
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
  const int wn = wave % WN, wm = wave / WN;
  const int rl = lane & 31, half = lane >> 5;

  const int2 tile = tile_of(p);
  const int n0 = tile.x * BN, m0 = tile.y * BM;

  // row and chunk of a lane in copy j: lane l fills slot l % 8 of row l / 8;
  // chunk c of a row lies in slot c ^ ((row >> 1) & 7) (reads of 16 rows at
  // one chunk then touch all banks)
  const uint8_t *wsrc = p.w + (int64_t)n0 * p.w_ld;
  const uint8_t *xsrc = p.x + (int64_t)m0 * p.x_ld;
  uint32_t won[NC], xom[MC];
  const int chunk_e = (lane & 7) ^ (lane >> 4);  // even row groups; odd ones: ^ 4
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int g = wave * NC + j, row = g * 8 + (lane >> 3);
    won[j] = (uint32_t)min(row, p.n - 1 - n0) * (uint32_t)p.w_ld + (chunk_e ^ ((g & 1) * 4)) * 16;
  }
#pragma unroll
  for (int j = 0; j < MC; ++j) {
    const int g = wave * MC + j, row = g * 8 + (lane >> 3);
    xom[j] = (uint32_t)min(row, p.m - 1 - m0) * (uint32_t)p.x_ld + (chunk_e ^ ((g & 1) * 4)) * 16;
  }
  // the group's tiles [t0, t1); every group takes `rounds` steps of the loop
  const int steps = (p.k + kBK - 1) / kBK, full = p.k / kBK;
  const int t0 = steps * group / KS, t1 = steps * (group + 1) / KS;
  const int rounds = (steps + KS - 1) / KS;
  auto load = [&](int t) {
    const uint32_t dst = lds0 + (uint32_t)(t % STAGES) * STAGE;
    const int k0 = t * kBK;
    if (t < full) {
#pragma unroll
      for (int j = 0; j < NC; ++j) copy1(wsrc + k0, won[j], dst + (wave * NC + j) * 1024);
#pragma unroll
      for (int j = 0; j < MC; ++j)
        copy1(xsrc + k0, xom[j], dst + BN * kBK + (wave * MC + j) * 1024);
    } else {
      // chunks past k: zeros for x, so that they count nothing whatever w's hold
      // there; the stage's last readers are behind the barrier as for a copy
#pragma unroll
      for (int j = 0; j < NC; ++j)
        if (k0 + (chunk_e ^ (((wave * NC + j) & 1) * 4)) * 16 < p.k)
          copy1(wsrc + k0, won[j], dst + (wave * NC + j) * 1024);
#pragma unroll
      for (int j = 0; j < MC; ++j) {
        const uint32_t at = BN * kBK + (wave * MC + j) * 1024;
        if (k0 + (chunk_e ^ (((wave * MC + j) & 1) * 4)) * 16 < p.k)
          copy1(xsrc + k0, xom[j], dst + at);
        else
          *(lds_u32x4_t *)(lds + (t % STAGES) * STAGE + at + lane * 16) = u32x4_t{0u, 0u, 0u, 0u};
      }
    }
  };

  i32x16_t acc[TN][TM] = {};
  const int swz = (rl >> 1) & 7;  // (rows of a fragment start at multiples of 32)
  const lds_u8_t *const wrow = lds + (wn * TN * 32 + rl) * kBK;
  const lds_u8_t *const xrow = lds + BN * kBK + (wm * TM * 32 + rl) * kBK;
  auto compute = [&](int t) {
    const uint32_t st = (uint32_t)(t % STAGES) * STAGE;
    i32x4_t wf[2][TN], xf[2][TM];
    auto read = [&](int s) {
      const uint32_t c = (uint32_t)(((2 * s + half) ^ swz) << 4) + st;
#pragma unroll
      for (int i = 0; i < TN; ++i)
        wf[s & 1][i] = __builtin_bit_cast(i32x4_t, *(const lds_u32x4_t *)(wrow + c + i * 32 * kBK));
#pragma unroll
      for (int i = 0; i < TM; ++i)
        xf[s & 1][i] = __builtin_bit_cast(i32x4_t, *(const lds_u32x4_t *)(xrow + c + i * 32 * kBK));
    };
    read(0);
#pragma unroll
    for (int s = 0; s < kBK / 32; ++s) {
      if (s + 1 < kBK / 32) read(s + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[s & 1][i], xf[s & 1][j], acc[i][j],
                                                            0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i)
    if (t0 + i < t1) load(t0 + i);
  for (int i = 0; i < rounds; ++i) {
    const int t = t0 + i;
    // this tile's own copies have landed (those of later whole tiles may be
    // under way); the barrier makes every wave's visible and the stage of the
    // tile before free
    if (STAGES > 2 && t + STAGES - 2 < min(t1, full))
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * (NC + MC)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t + STAGES - 1 < t1) load(t + STAGES - 1);
    if (KS == 1 || t < t1) compute(t);
  }

  // ---- epilogue: out = acc xs ws + bias, rounded to bf16 through LDS so that
  // rows are stored whole
  __syncthreads();
  join_sums<KS, WAVES>(all, acc, group, wave * 64 + lane);
  store_tile<TN, TM, BN, THREADS>(p, all, acc, n0, m0, wn, wm, wave, group == 0);
}

// WN x WM x KG waves, each TN x TM products of 32 x 32 over its KG-th part of a
// tile's k.  One ring of tiles for the workgroup; a wave reads its fragments of
// tile t + 1 and copies its part of tile t + STAGES - 1 between the products of
// tile t, so that neither LDS, nor the copies' issue, nor the barrier stands between
// two products.  A CU alone takes 0.34 us per 128 x 128 x 128 so (0.21 at the matrix
// units' rate), where rings whose waves copy, read and then multiply take 0.48 with
// eight waves and 0.57 with four: waiting for memory was none of it (the same with
// every byte in L2 and with 2 to 5 stages).  Tiles of 64 x 64 take 256 bytes of k at
// a time, half the barriers: 200 x 4096 x 4096 9.4 against 10.7 us.
template <int WN, int WM, int TN, int TM, int STAGES, int KG, int BK>
__global__ __launch_bounds__(WN *WM *KG * 64) void gemm_pipe_kernel(GemmParams p) {
  constexpr int WAVES = WN * WM * KG, THREADS = WAVES * 64;
  constexpr int NS = BK / 32 / KG;  // fragments of a tile that a wave reads
  constexpr int BN = WN * TN * 32, BM = WM * TM * 32;
  constexpr int CPR = BK / 16, RPC = 64 / CPR;  // chunks per row, rows per copy
  // copies of a tile and per wave; where they are no multiple of the waves, the last
  // ones are made again (the same bytes to the same place)
  constexpr int CN = BN / RPC, CM = BM / RPC;
  constexpr int NC = (CN + WAVES - 1) / WAVES, MC = (CM + WAVES - 1) / WAVES;
  static_assert(BN % RPC == 0 && BM % RPC == 0, "whole copies");
  static_assert(NS >= 2 && STAGES >= 3, "read and copied ahead");
  constexpr int STAGE = (BN + BM) * BK;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x;
  const int wave = readfirstlane(tid >> 6);
  const int lane = tid & 63;
  lds_u8_t *const lds = (lds_u8_t *)smem;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
  const int wn = wave % WN, wm = wave / WN % WM, group = wave / (WN * WM);
  const int rl = lane & 31, half = lane >> 5;

  const int2 tile = tile_of(p);
  const int n0 = tile.x * BN, m0 = tile.y * BM;
  const uint8_t *wsrc = p.w + (int64_t)n0 * p.w_ld;
  const uint8_t *xsrc = p.x + (int64_t)m0 * p.x_ld;
  uint32_t won[NC], xom[MC];
  // chunk c of a row lies in slot c ^ swz(row): reads of 16 rows at one chunk touch
  // all banks
  auto swz = [](int row) { return BK == 128 ? (row >> 1) & 7 : row & 15; };
  // row and chunk of the lane in copy g of an operand
  const int crow = lane / CPR;
  auto chunk = [&](int g) { return (lane % CPR) ^ swz(g * RPC + crow); };
  auto nth = [&](int j) {  // the wave's copy j: its number in W (X)
    if (j < NC) return CN % WAVES ? min(wave * NC + j, CN - 1) : wave * NC + j;
    return CM % WAVES ? min(wave * MC + j - NC, CM - 1) : wave * MC + j - NC;
  };
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int g = nth(j);
    won[j] = (uint32_t)min(g * RPC + crow, p.n - 1 - n0) * (uint32_t)p.w_ld + chunk(g) * 16;
  }
#pragma unroll
  for (int j = 0; j < MC; ++j) {
    const int g = nth(NC + j);
    xom[j] = (uint32_t)min(g * RPC + crow, p.m - 1 - m0) * (uint32_t)p.x_ld + chunk(g) * 16;
  }
  const int steps = (p.k + BK - 1) / BK, full = p.k / BK;
  // copy j of tile t, to the stage at dst
  auto copy = [&](int t, uint32_t dst, int j) {
    if (j < NC)
      copy1(wsrc + t * BK, won[j], lds0 + dst + nth(j) * 1024);
    else
      copy1(xsrc + t * BK, xom[j - NC], lds0 + dst + BN * BK + nth(j) * 1024);
  };
  // the last tile where k ends inside it: chunks past k are zeros for x, so that
  // they count nothing whatever w's hold there
  auto load_part = [&](int t, uint32_t dst) {
    const int k0 = t * BK;
#pragma unroll
    for (int j = 0; j < NC + MC; ++j) {
      const int g = nth(j);
      if (k0 + chunk(g) * 16 < p.k)
        copy(t, dst, j);
      else if (j >= NC)
        *(lds_u32x4_t *)(lds + dst + BN * BK + g * 1024 + lane * 16) = u32x4_t{0u, 0u, 0u, 0u};
    }
  };

  i32x16_t acc[TN][TM] = {};
  const int mine = swz(rl);  // (rows of a fragment start at multiples of 32)
  const lds_u8_t *const wrow = lds + (wn * TN * 32 + rl) * BK;
  const lds_u8_t *const xrow = lds + BN * BK + (wm * TM * 32 + rl) * BK;
  i32x4_t wf[NS][TN], xf[NS][TM];
  auto read = [&](uint32_t st, int s) {
    const uint32_t c = (uint32_t)(((2 * (group * NS + s) + half) ^ mine) << 4) + st;
#pragma unroll
    for (int i = 0; i < TN; ++i)
      wf[s][i] = __builtin_bit_cast(i32x4_t, *(const lds_u32x4_t *)(wrow + c + i * 32 * BK));
#pragma unroll
    for (int i = 0; i < TM; ++i)
      xf[s][i] = __builtin_bit_cast(i32x4_t, *(const lds_u32x4_t *)(xrow + c + i * 32 * BK));
  };
  auto multiply = [&](int s) {  // (in its place: reads before it, copies after it)
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[s][i], xf[s][j], acc[i][j], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i)
    if (i < full) {
#pragma unroll
      for (int j = 0; j < NC + MC; ++j) copy(i, i * STAGE, j);
    } else if (i < steps) {
      load_part(i, i * STAGE);
    }
  if (STAGES - 1 <= full)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * (NC + MC)) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  uint32_t st = 0, prev = (STAGES - 1) * STAGE;  // stages of this tile and of the one before
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) read(0, s);
  for (int t = 0; t < steps; ++t) {
    // tile t - 1 + STAGES goes to the stage that tile t - 1 left
    const int next = t - 1 + STAGES;
    const bool whole = next < full;
    auto some = [&](int c) {
      if (whole) {
#pragma unroll
        for (int j = 0; j < NC + MC; ++j)
          if (j * NS / (NC + MC) == c) copy(next, prev, j);
      }
    };
    const uint32_t following = st + STAGE == STAGES * STAGE ? 0 : st + STAGE;
    read(st, NS - 1);
    multiply(0);
    // tile t + 1 has landed, and every wave has read tile t - 1 (past the last
    // tile what is read counts nothing)
    if (next - 1 < full)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 3) * (NC + MC)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if (s + 1 < NS) {
        read(following, s);
        multiply(s + 1);
      }
      some(s);
      if (s == 0 && !whole && next < steps) {
        load_part(next, prev);
        __builtin_amdgcn_s_waitcnt(0xC07F);
      }
    }
    prev = st, st = following;
  }
  __syncthreads();
  join_sums<KG, WN * WM>(lds, acc, group, wave % (WN * WM) * 64 + lane);
  store_tile<TN, TM, BN, THREADS>(p, lds, acc, n0, m0, wn, wm, wave, group == 0);
}

// Tiles of 256 x 256 by eight waves in two groups that take turns: while one
// group's waves issue their 16 products, the other's (one of each to a SIMD) read
// their fragments and copy a tile ahead, so that the matrix units do not wait for
// LDS, copies or barriers.  Four stages of 64 bytes of k.
template <int WN, int WM, int TN, int TM>
__global__ __launch_bounds__(WN *WM * 64) void gemm_turns_kernel(GemmParams p) {
  constexpr int WAVES = WN * WM, STAGES = 4, BK = 64;
  constexpr int BN = WN * TN * 32, BM = WM * TM * 32;
  constexpr int NC = BN / 16 / WAVES, MC = BM / 16 / WAVES;  // copies per wave and tile
  static_assert(BN % (16 * WAVES) == 0 && BM % (16 * WAVES) == 0, "whole copies");
  constexpr int STAGE = (BN + BM) * BK;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  lds_u8_t *const lds = (lds_u8_t *)smem;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
  const int tid = threadIdx.x;
  const int wave = readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int wn = wave % WN, wm = wave / WN;
  const int rl = lane & 31, half = lane >> 5;
  const int2 tile = tile_of(p);
  const int n0 = tile.x * BN, m0 = tile.y * BM;

  // lane l of a copy fills slot l % 4 of row l / 4; chunk c of a row lies in slot
  // c ^ ((row >> 2) & 3)
  const uint8_t *wsrc = p.w + (int64_t)n0 * p.w_ld;
  const uint8_t *xsrc = p.x + (int64_t)m0 * p.x_ld;
  const int chunk = (lane & 3) ^ ((lane >> 4) & 3);
  uint32_t won[NC], xom[MC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int row = (wave * NC + j) * 16 + (lane >> 2);
    won[j] = (uint32_t)min(row, p.n - 1 - n0) * (uint32_t)p.w_ld + chunk * 16;
  }
#pragma unroll
  for (int j = 0; j < MC; ++j) {
    const int row = (wave * MC + j) * 16 + (lane >> 2);
    xom[j] = (uint32_t)min(row, p.m - 1 - m0) * (uint32_t)p.x_ld + chunk * 16;
  }
  const int steps = (p.k + BK - 1) / BK, full = p.k / BK;
  auto load = [&](int t) {
    const uint32_t st = (uint32_t)(t % STAGES) * STAGE;
    const int k0 = t * BK;
    auto copies = [&]() {
#pragma unroll
      for (int j = 0; j < NC; ++j) copy1(wsrc + k0, won[j], lds0 + st + (wave * NC + j) * 1024);
#pragma unroll
      for (int j = 0; j < MC; ++j)
        copy1(xsrc + k0, xom[j], lds0 + st + BN * BK + (wave * MC + j) * 1024);
    };
    if (t < full) {
      copies();
    } else if (k0 + chunk * 16 < p.k) {
      copies();
    } else {
      // chunks past k: zeros for x, so that they count nothing whatever w's hold
#pragma unroll
      for (int j = 0; j < MC; ++j)
        *(lds_u32x4_t *)(lds + st + BN * BK + (wave * MC + j) * 1024 + lane * 16) =
            u32x4_t{0u, 0u, 0u, 0u};
    }
  };

  i32x16_t acc[TN][TM] = {};
  const int swz = (rl >> 2) & 3;
  const lds_u8_t *const wrow = lds + (wn * TN * 32 + rl) * BK;
  const lds_u8_t *const xrow = lds + BN * BK + (wm * TM * 32 + rl) * BK;
  i32x4_t wf[2][TN], xf[2][TM];
  auto read = [&](int t, int s) {
    const uint32_t c = (uint32_t)(((2 * s + half) ^ swz) << 4) + (uint32_t)(t % STAGES) * STAGE;
#pragma unroll
    for (int i = 0; i < TN; ++i)
      wf[s][i] = __builtin_bit_cast(i32x4_t, *(const lds_u32x4_t *)(wrow + c + i * 32 * BK));
#pragma unroll
    for (int i = 0; i < TM; ++i)
      xf[s][i] = __builtin_bit_cast(i32x4_t, *(const lds_u32x4_t *)(xrow + c + i * 32 * BK));
  };
  auto multiply = [&](int s) {
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int i = 0; i < TN; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[s][i], xf[s][j], acc[i][j], 0, 0, 0);
  };
  auto barrier = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  };
#pragma unroll
  for (int t = 0; t < STAGES - 1; ++t)
    if (t < steps) load(t);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  barrier();
  // the second group runs one barrier behind the first: in step t a group copies
  // into the stage of tile t - 1, which the other has read before its last
  // barrier, and waits for its own copies of tile t + 1, so that two barriers on
  // both groups' have landed
  const bool second = wave >= WAVES / 2;
  if (second) barrier();
  for (int t = 0; t < steps; ++t) {
    read(t, 0);
    read(t, 1);
    if (t + 3 < steps) load(t + 3);
    if (t + 3 < full)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * (NC + MC)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    barrier();
    __builtin_amdgcn_s_setprio(1);
    multiply(0);
    multiply(1);
    __builtin_amdgcn_s_setprio(0);
    barrier();
  }
  if (!second) barrier();
  __syncthreads();
  store_tile<TN, TM, BN, WAVES * 64>(p, lds, acc, n0, m0, wn, wm, wave, true);
}
// Streaming form, at most 16 rows: a workgroup takes 16 columns, its waves
// shares of k, operands straight from memory (v_mfma_i32_16x16x64_i8).
constexpr int kStreamWaves = 8;
constexpr int kStreamAhead = 4;  // k steps loaded together

__global__ __launch_bounds__(kStreamWaves * 64) void stream_kernel(GemmParams p) {
  __shared__ int red[kStreamWaves][16][17];
  const int tid = threadIdx.x;
  const int wave = readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int steps = (p.k + 63) / 64;
  const int s0 = steps * wave / kStreamWaves, s1 = steps * (wave + 1) / kStreamWaves;
  const uint8_t *wp = p.w + (int64_t)min(n0 + r, p.n - 1) * p.w_ld;
  const uint8_t *xp = p.x + (int64_t)min(r, p.m - 1) * p.x_ld;
  i32x4_t acc = {};
  constexpr int U = kStreamAhead;
  for (int s = s0; s < s1; s += U) {
    i32x4_t wf[U], xf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // past the share or k: a place that is there, cleared below
      const int k = min(s + u, s1 - 1) * 64 + g * 16;
      const int kk = k < p.k ? k : 0;
      wf[u] = *reinterpret_cast<const i32x4_t *>(wp + kk);
      xf[u] = *reinterpret_cast<const i32x4_t *>(xp + kk);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = s + u < s1 && (s + u) * 64 + g * 16 < p.k;
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], in ? xf[u] : i32x4_t{0, 0, 0, 0}, acc, 0,
                                                  0, 0);
    }
  }
  // lane (r, g): column (token) r, rows (channels) 4 g ..
#pragma unroll
  for (int e = 0; e < 4; ++e) red[wave][g * 4 + e][r] = acc[e];
  __syncthreads();
  const int c = tid % 16, t = tid / 16;
  if (t >= p.m || n0 + c >= p.n) return;
  int v = 0;
#pragma unroll
  for (int i = 0; i < kStreamWaves; ++i) v += red[i][c][t];
  const float y = fmaf((float)v * p.xs[t], p.ws[n0 + c], bias_at(p, n0 + c));
  p.out[(int64_t)t * p.out_ld + n0 + c] = (uint16_t)(pack2_bf16(y, 0.f) & 0xffffu);
}

// (a grid of 2^32 threads and more would be cut without an error)
int check_grid(int64_t groups, int threads) {
  if (groups * threads < (1ll << 32)) return MIA_OK;
  return set_error(MIA_ERR_VALUE, "int8_linear: more tiles than a grid holds");
}

template <auto kernel>
int launch_tiles(const GemmParams &p, int threads, int bytes, hipStream_t s) {
  // (said once per device: the call takes a few us)
  static std::atomic<uint64_t> said{0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 64;
  if (bytes > 65536 && (dev >= 64 || !(said.load(std::memory_order_relaxed) >> dev & 1))) {
    const hipError_t e = hipFuncSetAttribute((const void *)kernel,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return check_hip(e, "int8_linear");
    if (dev < 64) said.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (const int rc = check_grid((int64_t)p.mt * p.nt, threads)) return rc;
  kernel<<<p.mt * p.nt, threads, bytes, s>>>(p);
  return check_hip(hipGetLastError(), "int8_linear");
}

template <int WN, int WM, int TN, int TM, int STAGES, int KS = 1>
int launch_gemm(GemmParams &p, hipStream_t s) {
  constexpr int BN = WN * TN * 32, BM = WM * TM * 32;
  p.nt = (p.n + BN - 1) / BN;
  p.mt = (p.m + BM - 1) / BM;
  constexpr int bytes = (BN + BM) * kBK * STAGES * KS;
  static_assert(bytes >= BN * 8 + WN * WM * KS * 32 * (TN * 64 + 16), "epilogue fits");
  static_assert(bytes >= join_bytes(KS, WN * WM, TN * TM), "sums fit");
  return launch_tiles<gemm_kernel<WN, WM, TN, TM, STAGES, KS>>(p, WN * WM * KS * 64, bytes, s);
}

template <int WN, int WM, int TN, int TM, int STAGES, int KG, int BK>
int launch_pipe(GemmParams &p, hipStream_t s) {
  constexpr int BN = WN * TN * 32, BM = WM * TM * 32;
  p.nt = (p.n + BN - 1) / BN;
  p.mt = (p.m + BM - 1) / BM;
  constexpr int bytes = (BN + BM) * BK * STAGES;
  static_assert(bytes >= BN * 8 + WN * WM * KG * 32 * (TN * 64 + 16), "epilogue fits");
  static_assert(bytes >= join_bytes(KG, WN * WM, TN * TM), "sums fit");
  return launch_tiles<gemm_pipe_kernel<WN, WM, TN, TM, STAGES, KG, BK>>(p, WN * WM * KG * 64, bytes, s);
}

int launch_turns(GemmParams &p, hipStream_t s) {
  p.nt = (p.n + 255) / 256;
  p.mt = (p.m + 255) / 256;
  return launch_tiles<gemm_turns_kernel<4, 2, 2, 4>>(p, 512, 512 * 64 * 4, s);
}

int launch_stream(GemmParams &p, hipStream_t s) {
  if (const int rc = check_grid(((int64_t)p.n + 15) / 16, kStreamWaves * 64)) return rc;
  stream_kernel<<<(p.n + 15) / 16, kStreamWaves * 64, 0, s>>>(p);
  return check_hip(hipGetLastError(), "int8_linear");
}

// The forms of the product: tile, workgroups that a CU holds, and the time of a
// call, once + rounds (round + step k / 128) us, where a round is a tile on
// every CU.  The constants are least squares over measurements at 1 to 8191 rows
// of k = 256 to 14336 and 512 to 10240 columns, weights rotated through 256 MB, of
// which the memory-side cache holds a part: weights from memory take longer, the
// fewer the rows the more, with the same forms ahead.  The form chosen by them took
// 0.3 % longer than the fastest one on the geometric mean, 22 % at most (8191 x 2880 x
// 5120: 155 against 127 us with a few weights in turn, 157 against 152 from memory; a
// clock that falls under load is no part of the model).  Heights of 160 and 192
// rows are for sizes that would take a round more at 128.  Examples, us, by form in
// the table's order, weights rotated through 1.6 GB; in brackets that of the form
// taken at 240 MB:
//   4 x 2048 x 2048, the last five: 9.1, 7.2, 5.4, 6.5, 3.9 (3.6)
//   16 x 4096 x 4096, the last five: 14.8, 10.7, 7.8, 9.9, 7.1 (6.4)
//   64 x 2880 x 5120, four before the last: 17.8, 12.1, 13.8, 10.8 (9.1)
//   64 x 4096 x 6144, four before the last: 17.8, 13.3, 14.7, 11.3 (8.1)
//   180 x 4096 x 4096: 52.6, 30.9, 26.0, 21.7, 19.8, 16.5, 12.2, 19.5, 17.7 (9.3)
//   517 x 2880 x 5120: 35.6, 23.6, 24.0, 20.6, 17.3, 27.7, 27.9, 62.5, 46.1 (18.0-19.7)
//   600 x 8192 x 10240, the first five: 89.8, 69.2, 93.4, 87.4, 76.8 (55.3)
//   850 x 4096 x 6144, the first five: 48.8, 33.9, 31.6, 44.0, 42.7 (29.1)
//   8191 x 2880 x 5120, the first five: 152, 157, 162, 178, 194 (156)
//   8191 x 8192 x 10240, the first five, 400 MB: 575-581, 679-698, 715-737, 764, 781
struct Form {
  int bm, bn, per_cu, rows;  // rows: at most (0: any number)
  float once, round, step;
  int (*launch)(GemmParams &, hipStream_t);
};
const Form kForms[] = {
    {256, 256, 1, 0, -15.0f, 22.2f, 1.149f, launch_turns},
    {128, 128, 2, 0, -6.5f, 10.3f, 0.685f, launch_gemm<2, 2, 2, 2, 2, 1>},
    {192, 128, 1, 0, -3.5f, 8.0f, 0.574f, launch_pipe<2, 6, 2, 1, 4, 1, 128>},
    {160, 128, 1, 0, -2.0f, 6.3f, 0.545f, launch_pipe<2, 5, 2, 1, 4, 1, 128>},
    {128, 128, 1, 0, -2.0f, 5.8f, 0.417f, launch_pipe<2, 4, 2, 1, 4, 1, 128>},
    {64, 128, 1, 0, -0.3f, 3.6f, 0.301f, launch_pipe<4, 2, 1, 1, 5, 1, 128>},
    {64, 64, 1, 0, 0.5f, 2.9f, 0.188f, launch_pipe<2, 2, 1, 1, 5, 2, 256>},
    {32, 32, 1, 0, 1.4f, 1.8f, 0.113f, launch_gemm<1, 1, 1, 1, 3, 4>},
    {32, 64, 1, 0, 0.9f, 2.4f, 0.139f, launch_gemm<2, 1, 1, 1, 3, 4>},
    {16, 16, 1, 16, 1.9f, 0.8f, 0.073f, launch_stream},
};

constexpr int64_t kMostGroups = 1 << 23;  // a grid's threads stay below 2^32

template <int LANES, int NV, bool NORM>
void launch_rows_form(const mia_quant_rows_args &a, hipStream_t s) {
  constexpr int RPB = 256 / LANES;
  const int64_t groups = (a.rows + RPB - 1) / RPB;
  // with gamma in registers as many workgroups as are resident at once
  constexpr int RESIDENT = NV == 1 ? 8 : NV == 2 ? 6 : NV == 4 ? 4 : 2;
  const int64_t most = NORM ? (int64_t)cu_count() * RESIDENT : kMostGroups;
  quant_rows_kernel<LANES, NV, NORM><<<(unsigned)std::min(groups, most), 256, 0, s>>>(a);
}

template <bool NORM>
void launch_rows(const mia_quant_rows_args &a, hipStream_t s) {
  if (a.dim <= 512) launch_rows_form<64, 1, NORM>(a, s);
  else if (a.dim <= 1024) launch_rows_form<64, 2, NORM>(a, s);
  else if (a.dim <= 2048) launch_rows_form<256, 1, NORM>(a, s);
  else if (a.dim <= 4096) launch_rows_form<256, 2, NORM>(a, s);
  else if (a.dim <= 8192) launch_rows_form<256, 4, NORM>(a, s);
  else launch_rows_form<256, 8, NORM>(a, s);
}

}  // namespace

int launch_quant_rows(const mia_quant_rows_args &a, hipStream_t s) {
  auto ok = [](const void *p, int64_t al) { return !p || (uintptr_t)p % al == 0; };
  const bool vec = a.dim % 8 == 0 && a.dim <= 16384 && a.x_stride % 8 == 0 &&
                   a.codes_stride % 8 == 0 && ok(a.x, 16) && ok(a.add0, 16) && ok(a.add1, 16) &&
                   ok(a.gamma, 16) && ok(a.codes, 8);
  if (!vec) quant_rows_any_kernel<<<(unsigned)std::min(a.rows, kMostGroups), 256, 0, s>>>(a);
  else if (a.norm) launch_rows<true>(a, s);
  else launch_rows<false>(a, s);
  return check_hip(hipGetLastError(), "quant_rows");
}

int int8_linear_forms() { return (int)(sizeof(kForms) / sizeof(kForms[0])); }

// The form that the measured costs say is the fastest.
int int8_linear_choice(const mia_int8_linear_args &a) {
  const float steps = (float)a.k / kBK;
  const int cus = cu_count();
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < int8_linear_forms(); ++i) {
    const Form &f = kForms[i];
    if (f.rows < a.rows && f.rows) continue;
    const int64_t tiles = (int64_t)((a.rows + f.bm - 1) / f.bm) * ((a.n + f.bn - 1) / f.bn);
    const int64_t rounds = (tiles + f.per_cu * cus - 1) / (f.per_cu * cus);
    const float cost = f.once + (float)rounds * (f.round + steps * f.step);
    if (i == 0 || cost < least) least = cost, best = i;
  }
  return best;
}

int launch_int8_linear(const mia_int8_linear_args &a, int form, hipStream_t s) {
  const Form &f = kForms[form];
  if (f.rows && f.rows < a.rows)
    return set_error(MIA_ERR_VALUE, "int8_linear: more rows than the form takes");
  GemmParams p = {};
  p.x = (const uint8_t *)a.x, p.w = (const uint8_t *)a.w;
  p.x_ld = a.rows == 1 ? 0 : a.x_stride, p.w_ld = a.n == 1 ? 0 : a.w_stride;
  p.xs = a.x_scales, p.ws = a.w_scales;
  p.bias = a.bias, p.bias_bf16 = a.bias_bf16;
  p.out = (uint16_t *)a.out, p.out_ld = a.out_stride;
  p.m = a.rows, p.n = a.n, p.k = a.k;
  p.vec = a.n % 8 == 0 && a.out_stride % 8 == 0 && (uintptr_t)a.out % 16 == 0;
  return f.launch(p, s);
}

}  // namespace mia
