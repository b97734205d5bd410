// quant_cache.hip — K/V rows quantised to 8 bits as they are written to the
// paged cache, with one fp32 scale per (token, kv head), and read back.
//
// Mathematics.  A row x[0..d) with amax = max |x| is stored as
//   scale = fl32(amax / Q),  code = rn(x * Q / amax),
// Q = 127 for int8 (ties to even) and 448 for e4m3fn, and read back as
// fl(code * scale).  Every code is the rounding of the exact quotient: x and
// amax are scaled by the power of two of amax (exact), x * Q is exact for
// bf16 and f16 sources (at most 18 bits), and the quotient a / b is formed as
// q + (a - b q) / b with one fma for the remainder.  For sources of p <= 11
// bits a quotient off a border between two codes is at least 2^-19 of itself
// away from it (2 a - (2 n + 1) b is a nonzero integer at the smaller of the
// two exponents), far more than the quotient's error of 2^-23, and a quotient
// on a border is a number of few bits, which the last fma gives exactly.  An
// fp32 source may take the neighbouring code where its quotient lies within
// 2^-22 of a border.  A row with a NaN or an infinity gets the scale NaN and
// zero codes; a row of zeros the scale 0; where Q * scale would overflow (the
// largest fp32 values) the scale is the next smaller number.
//
// Layout.  A row is read by LPR lanes with 16 bytes each (8 elements), the
// maximum goes over those lanes with xor shuffles, and each lane stores its 8
// codes; a thread takes K and V of its (token, head).  Bound by HBM for long
// calls: 16383 tokens of 8 heads, d = 128, bf16 to int8 25.9 us (3.9 TB/s of
// rows, codes and scales; a large device copy moves 4.9), read back 18.6 us
// (5.5 TB/s); 2048 tokens 6.4 us each way.  A step's few rows take a launch and
// three dependent loads: 3.4 and 2.6 us.  With K and V by separate threads the
// long calls took 28 and 23.6 us.
#include <algorithm>

#include "mia_device.h"
#include "mia_internal.h"

namespace mia {
namespace {

struct QuantKParams {
  const uint8_t *rows[2];  // K, V rows (write: source, read: destination)
  int64_t r_t[2], r_h[2], r_d[2];  // element strides
  const void *slots;
  int slot_dtype;
  uint8_t *cache[2];
  int64_t c_blk[2], c_h[2], c_t[2], c_d[2];
  float *scales[2];
  int64_t s_blk[2], s_h[2], s_t[2];
  uint32_t n_rows;  // tokens * kv heads
  int64_t n_slots;
  int d, bs;
  FastDiv h_div, bs_div;
};

MIA_DEV int64_t load_slot(const void *slots, int dtype, uint32_t t) {
  if (dtype == MIA_DTYPE_I64) return reinterpret_cast<const int64_t *>(slots)[t];
  if (dtype == MIA_DTYPE_I32) return reinterpret_cast<const int32_t *>(slots)[t];
  return reinterpret_cast<const uint32_t *>(slots)[t];
}

struct RowPos {
  uint32_t t, h;
  int64_t slot, blk, off;
};

// Workgroups of a launch lie in rows of at most kGridX: a grid of 2^32 threads
// or more along x is cut to its low 32 bits without an error, and 2^26 rows of
// 64 lanes are that many.
constexpr uint32_t kGridX = 1u << 23;
template <int LPR>
MIA_DEV uint32_t row_of() {
  return (blockIdx.y * gridDim.x + blockIdx.x) * (256 / LPR) + threadIdx.x / LPR;
}

// Row `row` of the call and its place in the cache (slot < 0: a sentinel).
MIA_DEV RowPos row_pos(const QuantKParams &p, uint32_t row) {
  RowPos r;
  r.t = fdiv(row, p.h_div);
  r.h = row - r.t * p.h_div.d;
  r.slot = load_slot(p.slots, p.slot_dtype, r.t);
  if (r.slot >= p.n_slots) r.slot = -1;
  if (r.slot < 0) {
    r.blk = r.off = 0;
  } else if (p.n_slots <= 0x7fffffff) {
    r.blk = fdiv((uint32_t)r.slot, p.bs_div);
    r.off = r.slot - r.blk * p.bs;
  } else {
    r.blk = r.slot / p.bs;
    r.off = r.slot - r.blk * p.bs;
  }
  return r;
}

template <int SRC>
MIA_DEV float load_elem(const uint8_t *p, int64_t i) {
  if constexpr (SRC == MIA_DTYPE_BF16)
    return bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(p)[i]);
  else if constexpr (SRC == MIA_DTYPE_F16)
    return f16_bits_to_f32(reinterpret_cast<const uint16_t *>(p)[i]);
  else
    return reinterpret_cast<const float *>(p)[i];
}

template <int DST>
MIA_DEV uint32_t to_bits16(float x) {
  if constexpr (DST == MIA_DTYPE_BF16) return pack2_bf16(x, 0.f) & 0xffffu;
  else return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x);
}

// 8 elements from channel c0 of a row; channels at or past d are 0.
template <int SRC, bool VEC>
MIA_DEV void load8(const uint8_t *row, int64_t sd, int c0, int d, float (&x)[8]) {
  if constexpr (VEC) {
    if constexpr (SRC == MIA_DTYPE_F32) {
      const f32x4_t a = *reinterpret_cast<const f32x4_t *>(row + (int64_t)c0 * 4);
      const f32x4_t b = *reinterpret_cast<const f32x4_t *>(row + (int64_t)c0 * 4 + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
    } else {
      const u32x4_t w = *reinterpret_cast<const u32x4_t *>(row + (int64_t)c0 * 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (SRC == MIA_DTYPE_BF16) {
          x[2 * i] = bf16lo(w[i]);
          x[2 * i + 1] = bf16hi(w[i]);
        } else {
          x[2 * i] = f16_bits_to_f32(w[i] & 0xffffu);
          x[2 * i + 1] = f16_bits_to_f32(w[i] >> 16);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c0 + i < d ? load_elem<SRC>(row, (c0 + i) * sd) : 0.f;
  }
}

// LPR lanes per row, 8 channels each (d <= 8 LPR); a thread takes its chunk of
// the K and of the V row, so that two loads are in flight and the slot is
// resolved once.  VEC: d is a multiple of 8, rows are contiguous and 16-byte
// (cache: 8-byte) aligned.
template <int SRC, bool I8, int LPR, bool VEC>
__global__ __launch_bounds__(256) void quant_write_kernel(QuantKParams p) {
  const uint32_t row = row_of<LPR>();
  const int c0 = (threadIdx.x % LPR) * 8;
  const bool in = row < p.n_rows;
  const RowPos r = row_pos(p, in ? row : 0);
  const bool act = c0 < p.d;
  constexpr int SB = SRC == MIA_DTYPE_F32 ? 4 : 2;
  constexpr float Q = I8 ? 127.0f : 448.0f;
  float x[2][8];
#pragma unroll
  for (int y = 0; y < 2; ++y) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[y][i] = 0.f;
    if (act)
      load8<SRC, VEC>(p.rows[y] + ((int64_t)r.t * p.r_t[y] + (int64_t)r.h * p.r_h[y]) * SB,
                      p.r_d[y], c0, p.d, x[y]);
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    // maximum of the magnitudes as integers: an infinity or NaN is the largest
    uint32_t mag = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mag = max(mag, __float_as_uint(x[y][i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) mag = max(mag, (uint32_t)__shfl_xor((int)mag, o, 64));
    if (!in || r.slot < 0) continue;
    const float amax = __uint_as_float(mag);
    const bool bad = mag >= 0x7f800000u;
    const bool zero = bad || mag == 0;
    const int e = __builtin_amdgcn_frexp_expf(amax);
    const float b = zero ? 1.0f : ldexpf(amax, -e);  // [0.5, 1)
    float rc = __builtin_amdgcn_rcpf(b);
    rc = fmaf(fmaf(-b, rc, 1.0f), rc, rc);
    float y8[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = (zero ? 0.f : ldexpf(x[y][i], -e)) * Q;
      const float q = a * rc;
      y8[i] = fmaf(fmaf(-b, q, a), rc, q);
    }
    u32x2_t w;
    if constexpr (I8) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v |= ((uint32_t)(int)rintf(y8[4 * g + i]) & 0xffu) << (8 * i);
        w[g] = v;
      }
    } else {
      w[0] = e4m3fn_x4(y8[0], y8[1], y8[2], y8[3]);
      w[1] = e4m3fn_x4(y8[4], y8[5], y8[6], y8[7]);
    }
    uint8_t *dst = p.cache[y] + r.blk * p.c_blk[y] + (int64_t)r.h * p.c_h[y] + r.off * p.c_t[y];
    if constexpr (VEC) {
      if (act) *reinterpret_cast<u32x2_t *>(dst + c0) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < p.d)
          dst[(int64_t)(c0 + i) * p.c_d[y]] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
    if (threadIdx.x % LPR == 0) {
      float sc = amax / Q;
      // the largest fp32 values: code Q must not read back as an infinity
      if (SRC == MIA_DTYPE_F32 && sc * Q > 3.402823466e38f)
        sc = __uint_as_float(__float_as_uint(sc) - 1u);
      p.scales[y][r.blk * p.s_blk[y] + (int64_t)r.h * p.s_h[y] + r.off * p.s_t[y]] =
          bad ? __uint_as_float(0x7fc00000u) : sc;
    }
  }
}

template <int DST, bool I8, int LPR, bool VEC>
__global__ __launch_bounds__(256) void quant_read_kernel(QuantKParams p) {
  const uint32_t row = row_of<LPR>();
  const int c0 = (threadIdx.x % LPR) * 8;
  if (row >= p.n_rows || c0 >= p.d) return;
  const RowPos r = row_pos(p, row);
  uint32_t w[2][2] = {{0u, 0u}, {0u, 0u}};
  float s[2] = {0.f, 0.f};
  if (r.slot >= 0) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const uint8_t *src =
          p.cache[y] + r.blk * p.c_blk[y] + (int64_t)r.h * p.c_h[y] + r.off * p.c_t[y];
      s[y] = p.scales[y][r.blk * p.s_blk[y] + (int64_t)r.h * p.s_h[y] + r.off * p.s_t[y]];
      if constexpr (VEC) {
        const u32x2_t v = *reinterpret_cast<const u32x2_t *>(src + c0);
        w[y][0] = v[0];
        w[y][1] = v[1];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c0 + i < p.d)
            w[y][i >> 2] |= (uint32_t)src[(int64_t)(c0 + i) * p.c_d[y]] << (8 * (i & 3));
      }
    }
  }
  constexpr int DB = DST == MIA_DTYPE_F32 ? 4 : 2;
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t byte = (w[y][i >> 2] >> (8 * (i & 3))) & 0xffu;
      x[i] = (I8 ? (float)(int8_t)byte : e4m3fn_bits_to_f32(byte)) * s[y];
      // the product is rounded to fp32 in every case (an f16 result would
      // otherwise be formed by one mixed multiply, rounded once)
      if constexpr (DST == MIA_DTYPE_F16) asm("" : "+v"(x[i]));
    }
    uint8_t *dst = const_cast<uint8_t *>(p.rows[y]) +
                   ((int64_t)r.t * p.r_t[y] + (int64_t)r.h * p.r_h[y]) * DB;
    if constexpr (VEC) {
      if constexpr (DST == MIA_DTYPE_F32) {
        *reinterpret_cast<f32x4_t *>(dst + c0 * 4) = f32x4_t{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4_t *>(dst + c0 * 4 + 16) = f32x4_t{x[4], x[5], x[6], x[7]};
      } else {
        u32x4_t o;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o[i] = to_bits16<DST>(x[2 * i]) | (to_bits16<DST>(x[2 * i + 1]) << 16);
        *reinterpret_cast<u32x4_t *>(dst + c0 * 2) = o;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (c0 + i >= p.d) break;
        const int64_t o = (int64_t)(c0 + i) * p.r_d[y];
        if constexpr (DST == MIA_DTYPE_F32) reinterpret_cast<float *>(dst)[o] = x[i];
        else reinterpret_cast<uint16_t *>(dst)[o] = (uint16_t)to_bits16<DST>(x[i]);
      }
    }
  }
}

bool vec_ok(const mia_quant_kv_args &a) {
  const int64_t eb = a.row_dtype == MIA_DTYPE_F32 ? 4 : 2;
  auto rows = [&](const void *p, const int64_t *s) {
    return (uintptr_t)p % 16 == 0 && s[2] == 1 && s[0] * eb % 16 == 0 && s[1] * eb % 16 == 0;
  };
  auto pool = [&](const void *p, const int64_t *s) {
    return (uintptr_t)p % 8 == 0 && s[3] == 1 && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
  };
  return a.head_dim % 8 == 0 && rows(a.k, a.k_stride) && rows(a.v, a.v_stride) &&
         pool(a.k_cache, a.k_cache_stride) && pool(a.v_cache, a.v_cache_stride);
}

QuantKParams kparams(const mia_quant_kv_args &a) {
  QuantKParams p;
  const void *rows[2] = {a.k, a.v};
  const int64_t *rs[2] = {a.k_stride, a.v_stride};
  void *pools[2] = {a.k_cache, a.v_cache};
  const int64_t *cs[2] = {a.k_cache_stride, a.v_cache_stride};
  float *sc[2] = {a.k_scales, a.v_scales};
  const int64_t *ss[2] = {a.k_scale_stride, a.v_scale_stride};
  for (int y = 0; y < 2; ++y) {
    p.rows[y] = (const uint8_t *)rows[y];
    p.r_t[y] = rs[y][0], p.r_h[y] = rs[y][1], p.r_d[y] = rs[y][2];
    p.cache[y] = (uint8_t *)pools[y];
    p.c_blk[y] = cs[y][0], p.c_h[y] = cs[y][1], p.c_t[y] = cs[y][2], p.c_d[y] = cs[y][3];
    p.scales[y] = sc[y];
    p.s_blk[y] = ss[y][0], p.s_h[y] = ss[y][1], p.s_t[y] = ss[y][2];
  }
  p.slots = a.slots;
  p.slot_dtype = a.slot_dtype;
  p.n_rows = (uint32_t)(a.num_tokens * a.num_kv_heads);
  p.n_slots = (int64_t)a.num_blocks * a.block_size;
  p.d = a.head_dim;
  p.bs = a.block_size;
  p.h_div = make_fastdiv(a.num_kv_heads);
  p.bs_div = make_fastdiv(a.block_size);
  return p;
}

template <int DT, bool I8, int LPR, bool VEC>
void launch_one(const QuantKParams &p, bool write, hipStream_t s) {
  const uint32_t n = (p.n_rows + 256 / LPR - 1) / (256 / LPR), x = std::min(n, kGridX);
  const dim3 grid(x, (n + x - 1) / x);
  if (write) quant_write_kernel<DT, I8, LPR, VEC><<<grid, 256, 0, s>>>(p);
  else quant_read_kernel<DT, I8, LPR, VEC><<<grid, 256, 0, s>>>(p);
}

template <int DT, bool I8>
void launch_dtype(const QuantKParams &p, bool vec, bool write, hipStream_t s) {
  // rows of up to 64, 128, 256 and 512 channels
  if (!vec) launch_one<DT, I8, 64, false>(p, write, s);
  else if (p.d <= 64) launch_one<DT, I8, 8, true>(p, write, s);
  else if (p.d <= 128) launch_one<DT, I8, 16, true>(p, write, s);
  else launch_one<DT, I8, 64, true>(p, write, s);
}

}  // namespace

int launch_quant_kv(const mia_quant_kv_args &a, bool write, hipStream_t s) {
  const QuantKParams p = kparams(a);
  const bool vec = vec_ok(a);
  const bool i8 = a.code_dtype == MIA_DTYPE_I8;
  switch (a.row_dtype) {
    case MIA_DTYPE_BF16:
      i8 ? launch_dtype<MIA_DTYPE_BF16, true>(p, vec, write, s)
         : launch_dtype<MIA_DTYPE_BF16, false>(p, vec, write, s);
      break;
    case MIA_DTYPE_F16:
      i8 ? launch_dtype<MIA_DTYPE_F16, true>(p, vec, write, s)
         : launch_dtype<MIA_DTYPE_F16, false>(p, vec, write, s);
      break;
    default:
      i8 ? launch_dtype<MIA_DTYPE_F32, true>(p, vec, write, s)
         : launch_dtype<MIA_DTYPE_F32, false>(p, vec, write, s);
  }
  return check_hip(hipGetLastError(), write ? "quant_kv_write" : "quant_kv_read");
}

}  // namespace mia
