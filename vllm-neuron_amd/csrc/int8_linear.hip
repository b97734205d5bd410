// int8_linear.hip — rows quantised to int8 with one scale per token, and their
// product with int8 weights of one scale per output channel.
#include <algorithm>

#include "mia_device.h"
#include "mia_internal.h"

namespace mia {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) uint8_t lds_u8_t;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4_t;
typedef __attribute__((address_space(3))) u32x2_t lds_u32x2_t;
typedef __attribute__((address_space(3))) f32x4_t lds_f32x4_t;
typedef __attribute__((address_space(3))) float lds_f32_t;
typedef __attribute__((address_space(3))) uint16_t lds_u16_t;

// ---------------------------------------------------------------------------
// rows to int8
// ---------------------------------------------------------------------------
MIA_DEV float add_bf16(float a, float b) { return bf16lo(pack2_bf16(a + b, 0.f)); }

// The row's scale: fl32(amax / 127), of the normalised row.
MIA_DEV float row_scale(uint32_t mag, float ss, const mia_quant_rows_args &a) {
  if (mag >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  float amax = __uint_as_float(mag);
  if (a.norm) {
    const float n = (float)(a.dim_actual > 0 ? a.dim_actual : a.dim);
    amax *= 1.0f / sqrtf(ss / n + a.eps);
  }
  return amax / 127.0f;
}

MIA_DEV float gamma_at(const mia_quant_rows_args &a, int c) {
  if (a.gamma_bf16) return bf16_bits_to_f32(((const uint16_t *)a.gamma)[c]);
  return ((const float *)a.gamma)[c];
}

// LANES threads per row, NV vectors of 8 channels each, held in registers.
template <int LANES, int NV>
__global__ __launch_bounds__(256) void quant_rows_kernel(mia_quant_rows_args a) {
  constexpr int RPB = 256 / LANES;
  __shared__ float2 red[4];
  const int tid = threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LANES;
  const bool live = row < a.rows;
  const int64_t at = (live ? row : 0) * a.x_stride;
  float x[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * LANES + tid) * 8;
    u32x4_t w = {0u, 0u, 0u, 0u}, w0 = w, w1 = w;
    if (c < a.dim) {
      w = *reinterpret_cast<const u32x4_t *>((const uint16_t *)a.x + at + c);
      if (a.add0) w0 = *reinterpret_cast<const u32x4_t *>((const uint16_t *)a.add0 + at + c);
      if (a.add1) w1 = *reinterpret_cast<const u32x4_t *>((const uint16_t *)a.add1 + at + c);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[v][2 * i] = bf16lo(w[i]);
      x[v][2 * i + 1] = bf16hi(w[i]);
    }
    if (a.add0)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[v][2 * i] = add_bf16(x[v][2 * i], bf16lo(w0[i]));
        x[v][2 * i + 1] = add_bf16(x[v][2 * i + 1], bf16hi(w0[i]));
      }
    if (a.add1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[v][2 * i] = add_bf16(x[v][2 * i], bf16lo(w1[i]));
        x[v][2 * i + 1] = add_bf16(x[v][2 * i + 1], bf16hi(w1[i]));
      }
  }
  float ss = 0.f;
  if (a.norm) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[v][i], x[v][i], ss);
    if (a.gamma) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * LANES + tid) * 8;
        if (c >= a.dim) continue;
        if (a.gamma_bf16) {
          const u32x4_t g = *reinterpret_cast<const u32x4_t *>((const uint16_t *)a.gamma + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[v][2 * i] *= bf16lo(g[i]);
            x[v][2 * i + 1] *= bf16hi(g[i]);
          }
        } else {
          const f32x4_t g0 = *reinterpret_cast<const f32x4_t *>((const float *)a.gamma + c);
          const f32x4_t g1 = *reinterpret_cast<const f32x4_t *>((const float *)a.gamma + c + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[v][i] *= g0[i];
            x[v][4 + i] *= g1[i];
          }
        }
      }
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
    if (a.norm) ss += __shfl_xor(ss, o, 64);
  }
  if constexpr (LANES == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(__uint_as_float(mag), ss);
    __syncthreads();
    mag = max(max(__float_as_uint(red[0].x), __float_as_uint(red[1].x)),
              max(__float_as_uint(red[2].x), __float_as_uint(red[3].x)));
    ss = (red[0].y + red[1].y) + (red[2].y + red[3].y);
  }
  if (!live) return;
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
  if (tid == 0) a.scales[row] = row_scale(mag, ss, a);
}

// Any width, alignment and length: a workgroup per row, read twice.
__global__ __launch_bounds__(256) void quant_rows_any_kernel(mia_quant_rows_args a) {
  __shared__ float2 red[4];
  const int64_t row = blockIdx.x;
  const int64_t at = row * a.x_stride;
  float ss = 0.f;
  auto value = [&](int c, bool sum) {
    float x = bf16_bits_to_f32(((const uint16_t *)a.x)[at + c]);
    if (a.add0) x = add_bf16(x, bf16_bits_to_f32(((const uint16_t *)a.add0)[at + c]));
    if (a.add1) x = add_bf16(x, bf16_bits_to_f32(((const uint16_t *)a.add1)[at + c]));
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
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(__uint_as_float(mag), ss);
  __syncthreads();
  mag = max(max(__float_as_uint(red[0].x), __float_as_uint(red[1].x)),
            max(__float_as_uint(red[2].x), __float_as_uint(red[3].x)));
  ss = (red[0].y + red[1].y) + (red[2].y + red[3].y);
  RowCodes<127> rs;
  rs.set(mag);
  for (int c = threadIdx.x; c < a.dim; c += 256)
    ((uint8_t *)a.codes)[row * a.codes_stride + c] = (uint8_t)rs.int8(value(c, false));
  if (threadIdx.x == 0) a.scales[row] = row_scale(mag, ss, a);
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

// One 16-byte-per-lane copy HBM -> LDS: lane l's lands at lds_dst + 16 l.
// Inline assembly, so that the compiler adds no waits before reads of other
// stages; the wait for the copies is explicit.
MIA_DEV void copy1(const uint8_t *src, uint32_t off, uint32_t lds_dst) {
  const uint32_t m0 = readfirstlane((int)lds_dst);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, %1\n\t"
      :: "s"(m0), "s"(src), "v"(off) : "memory", "m0");
}

constexpr int kBK = 128;  // bytes of k per tile

// Tiled form.  WN x WM waves, each TN x TM products of 32 x 32.
template <int WN, int WM, int TN, int TM, int STAGES>
__global__ __launch_bounds__(WN *WM * 64) void gemm_kernel(GemmParams p) {
  constexpr int WAVES = WN * WM;
  constexpr int BN = WN * TN * 32, BM = WM * TM * 32;
  constexpr int NC = BN / 8 / WAVES, MC = BM / 8 / WAVES;  // copies per wave and tile
  static_assert(BN % (8 * WAVES) == 0 && BM % (8 * WAVES) == 0, "whole copies");
  constexpr int STAGE = (BN + BM) * kBK;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  lds_u8_t *const lds = (lds_u8_t *)smem;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;

  const int tid = threadIdx.x;
  const int wave = readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int wn = wave % WN, wm = wave / WN;
  const int rl = lane & 31, half = lane >> 5;

  // tiles: each XCD (workgroups go round robin over 8) takes a contiguous run
  // of them, in groups of 8 row tiles, so that its L2 holds what they share
  int tn, tm;
  {
    const int total = p.mt * p.nt;
    const int per = (total + 7) / 8;
    const int b = blockIdx.x;
    const int full = total / 8, rem = total % 8, xcd = b % 8;
    (void)per;
    const int id = xcd * full + min(xcd, rem) + b / 8;
    const int gsz = 8 * p.nt;
    const int g = id / gsz, first = g * 8, rows = min(p.mt - first, 8);
    const int r = id - g * gsz;
    tm = first + r % rows;
    tn = r / rows;
  }
  const int n0 = tn * BN, m0 = tm * BM;

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
  const int steps = (p.k + kBK - 1) / kBK, full = p.k / kBK;
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
      // chunks past k keep what the stage held: those of x are cleared below
#pragma unroll
      for (int j = 0; j < NC; ++j)
        if (k0 + (chunk_e ^ (((wave * NC + j) & 1) * 4)) * 16 < p.k)
          copy1(wsrc + k0, won[j], dst + (wave * NC + j) * 1024);
#pragma unroll
      for (int j = 0; j < MC; ++j)
        if (k0 + (chunk_e ^ (((wave * MC + j) & 1) * 4)) * 16 < p.k)
          copy1(xsrc + k0, xom[j], dst + BN * kBK + (wave * MC + j) * 1024);
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
  for (int t = 0; t < STAGES - 1; ++t)
    if (t < steps) load(t);
  for (int t = 0; t < steps; ++t) {
    // this tile's own copies have landed (those of later whole tiles may be
    // under way); the barrier makes every wave's visible and the stage of the
    // tile before free
    if (STAGES > 2 && t + STAGES - 2 < full)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * (NC + MC)) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t + STAGES - 1 < steps) load(t + STAGES - 1);
    if (t >= full) {
      // rows of x past k count nothing (whatever w's hold there)
      lds_u8_t *const xb = lds + (t % STAGES) * STAGE + BN * kBK;
      const int left = (p.k - t * kBK) / 16;
      for (int i = tid; i < BM * 8; i += WAVES * 64)
        if ((i & 7) >= left)
          *(lds_u32x4_t *)(xb + (i >> 3) * kBK + (((i & 7) ^ ((i >> 4) & 7)) << 4)) =
              u32x4_t{0u, 0u, 0u, 0u};
      __syncthreads();
    }
    compute(t);
  }

  // ---- epilogue: out = acc xs ws + bias, rounded to bf16 through LDS so that
  // rows are stored whole
  __syncthreads();
  lds_f32_t *const wsl = (lds_f32_t *)lds;  // [BN] scales, [BN] bias
  for (int i = tid; i < BN; i += WAVES * 64) {
    const int n = min(n0 + i, p.n - 1);
    wsl[i] = p.ws[n];
    wsl[BN + i] = bias_at(p, n);
  }
  __syncthreads();
  constexpr int ROWB = TN * 64 + 16;
  lds_u8_t *const stage = lds + BN * 8 + wave * 32 * ROWB;
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

// Streaming form, at most 16 MT rows: a workgroup takes 16 NT columns, its
// waves shares of k, operands straight from memory.
constexpr int kStreamWaves = 8;
constexpr int kStreamAhead = 4;  // k steps loaded together

template <int MT, int NT>
__global__ __launch_bounds__(kStreamWaves * 64) void stream_kernel(GemmParams p) {
  __shared__ __attribute__((aligned(16))) int red[kStreamWaves][NT * 16][MT * 16 + 1];
  const int tid = threadIdx.x;
  const int wave = readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * NT * 16;
  const int steps = (p.k + 63) / 64;
  const int s0 = steps * wave / kStreamWaves, s1 = steps * (wave + 1) / kStreamWaves;
  const uint8_t *wp[NT], *xp[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i) wp[i] = p.w + (int64_t)min(n0 + i * 16 + r, p.n - 1) * p.w_ld;
#pragma unroll
  for (int j = 0; j < MT; ++j) xp[j] = p.x + (int64_t)min(j * 16 + r, p.m - 1) * p.x_ld;
  i32x4_t acc[NT][MT] = {};
  constexpr int U = kStreamAhead;
  for (int s = s0; s < s1; s += U) {
    i32x4_t wf[U][NT], xf[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // past the share or k: a place that is there, cleared below
      const int k = min(s + u, s1 - 1) * 64 + g * 16;
      const int kk = k < p.k ? k : 0;
#pragma unroll
      for (int i = 0; i < NT; ++i) wf[u][i] = *reinterpret_cast<const i32x4_t *>(wp[i] + kk);
#pragma unroll
      for (int j = 0; j < MT; ++j) xf[u][j] = *reinterpret_cast<const i32x4_t *>(xp[j] + kk);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = s + u < s1 && (s + u) * 64 + g * 16 < p.k;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const i32x4_t b = in ? xf[u][j] : i32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NT; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][i], b, acc[i][j], 0, 0, 0);
      }
    }
  }
  // lane (r, g): column (token) r, rows (channels) 4 g ..
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][i * 16 + g * 4 + e][j * 16 + r] = acc[i][j][e];
  __syncthreads();
  for (int q = tid; q < NT * 16 * MT * 16; q += kStreamWaves * 64) {
    const int c = q % (NT * 16), t = q / (NT * 16);
    if (t >= p.m || n0 + c >= p.n) continue;
    int v = 0;
#pragma unroll
    for (int i = 0; i < kStreamWaves; ++i) v += red[i][c][t];
    const float y = fmaf((float)v * p.xs[t], p.ws[n0 + c], bias_at(p, n0 + c));
    p.out[(int64_t)t * p.out_ld + n0 + c] = (uint16_t)(pack2_bf16(y, 0.f) & 0xffffu);
  }
}

template <int WN, int WM, int TN, int TM, int STAGES>
int launch_gemm(GemmParams &p, hipStream_t s) {
  constexpr int BN = WN * TN * 32, BM = WM * TM * 32;
  p.nt = (p.n + BN - 1) / BN;
  p.mt = (p.m + BM - 1) / BM;
  constexpr int bytes = (BN + BM) * kBK * STAGES;
  static_assert(bytes >= BN * 8 + WN * WM * 32 * (TN * 64 + 16), "epilogue fits");
  auto kernel = gemm_kernel<WN, WM, TN, TM, STAGES>;
  if (bytes > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void *)kernel,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return check_hip(e, "int8_linear");
  }
  kernel<<<p.mt * p.nt, WN * WM * 64, bytes, s>>>(p);
  return check_hip(hipGetLastError(), "int8_linear");
}

}  // namespace

int launch_quant_rows(const mia_quant_rows_args &a, hipStream_t s) {
  auto ok = [](const void *p, int64_t al) { return !p || (uintptr_t)p % al == 0; };
  const bool vec = a.dim % 8 == 0 && a.dim <= 16384 && a.x_stride % 8 == 0 &&
                   a.codes_stride % 8 == 0 && ok(a.x, 16) && ok(a.add0, 16) && ok(a.add1, 16) &&
                   ok(a.gamma, 16) && ok(a.codes, 8);
  const unsigned rows = (unsigned)a.rows, rows4 = (unsigned)((a.rows + 3) / 4);
  if (!vec) quant_rows_any_kernel<<<rows, 256, 0, s>>>(a);
  else if (a.dim <= 512) quant_rows_kernel<64, 1><<<rows4, 256, 0, s>>>(a);
  else if (a.dim <= 1024) quant_rows_kernel<64, 2><<<rows4, 256, 0, s>>>(a);
  else if (a.dim <= 2048) quant_rows_kernel<256, 1><<<rows, 256, 0, s>>>(a);
  else if (a.dim <= 4096) quant_rows_kernel<256, 2><<<rows, 256, 0, s>>>(a);
  else if (a.dim <= 8192) quant_rows_kernel<256, 4><<<rows, 256, 0, s>>>(a);
  else quant_rows_kernel<256, 8><<<rows, 256, 0, s>>>(a);
  return check_hip(hipGetLastError(), "quant_rows");
}

int launch_int8_linear(const mia_int8_linear_args &a, hipStream_t s) {
  GemmParams p = {};
  p.x = (const uint8_t *)a.x, p.w = (const uint8_t *)a.w;
  p.x_ld = a.x_stride, p.w_ld = a.w_stride;
  p.xs = a.x_scales, p.ws = a.w_scales;
  p.bias = a.bias, p.bias_bf16 = a.bias_bf16;
  p.out = (uint16_t *)a.out, p.out_ld = a.out_stride;
  p.m = a.rows, p.n = a.n, p.k = a.k;
  p.vec = a.n % 8 == 0 && a.out_stride % 8 == 0 && (uintptr_t)a.out % 16 == 0;
  if (p.m <= 64) {
    const int c16 = (p.n + 15) / 16, c32 = (p.n + 31) / 32;
    if (p.m <= 16) stream_kernel<1, 1><<<c16, kStreamWaves * 64, 0, s>>>(p);
    else if (p.m <= 32) stream_kernel<2, 1><<<c16, kStreamWaves * 64, 0, s>>>(p);
    else stream_kernel<4, 2><<<c32, kStreamWaves * 64, 0, s>>>(p);
    return check_hip(hipGetLastError(), "int8_linear");
  }
  const int64_t big = (int64_t)((p.n + 255) / 256) * ((p.m + 255) / 256);
  if (big >= 192) return launch_gemm<4, 2, 2, 4, 2>(p, s);
  return launch_gemm<2, 2, 2, 2, 2>(p, s);
}

}  // namespace mia
