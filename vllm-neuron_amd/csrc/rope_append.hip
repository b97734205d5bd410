// rope_append.hip — Q and K rotated by positions on one to four axes, K and V
// appended to the paged cache in the same pass.
//
// Mathematics.  Channel pair i of the first R channels turns by pos[axis(i)] inv[i]:
// (x, y) -> (x cos - y sin, y cos + x sin), pairs (i, i + R / 2) or (2 i, 2 i + 1); the
// other channels pass.  Before it, where asked, each head's RMS norm.  K and V rows
// go to the slot's place as bf16, as e4m3 with a static scale per head, or as int8 or e4m3
// codes with the scale of their own maximum.  All in fp32 from the loaded bf16 to
// the stored value, rounded once; angles in 64 bits down to a fraction of a turn.
//
// A token's cosines and sines are computed once for its heads (R / 2 of them in LDS);
// a lane holds 8 channels, both members of each of its pairs, so that a rotation
// takes no exchange, and a head row lies in 8, 16 or 32 lanes, which reduce norm and
// maximum among themselves.  Bound by HBM: every value is read and written once.
// 16383 tokens of 32 + 8 + 8 heads, d = 128, 75 us (403 MB, 5.4 TB/s; a large copy moves
// 4.97); 2047 tokens of 48 + 8 + 8 heads with norms 16.2 us (67 MB, 4.1 TB/s: 2047
// workgroups' start); a decode step's 8 tokens to an int8 cache 4.5 us, launch
// and the chain position, angle, row.
#include <algorithm>

#include "mia_device.h"
#include "mia_internal.h"

namespace mia {
namespace {

enum AppendKind { kRows = 0, kBf16 = 1, kFp8Static = 2, kFp8 = 3, kI8 = 4 };

MIA_DEV int64_t load_int(const void *p, int dtype, int64_t i) {
  if (dtype == MIA_DTYPE_I64) return ((const int64_t *)p)[i];
  if (dtype == MIA_DTYPE_U32) return (int64_t)((const uint32_t *)p)[i];
  return (int64_t)((const int32_t *)p)[i];
}

// Axis of channel pair i: contiguous blocks of pairs, or the axes in turn while
// their pairs last (the rest to axis 0).
MIA_DEV int axis_of(const mia_rope_append_args &a, int i) {
  if (a.section_cycle) {
    const int x = i % a.axes;
    int n = a.section[0];
#pragma unroll
    for (int k = 1; k < 4; ++k) n = x == k ? a.section[k] : n;
    return i < n * a.axes ? x : 0;
  }
  int x = 0, end = a.section[0];
#pragma unroll
  for (int k = 1; k < 4; ++k) {
    if (k < a.axes && i >= end) x = k;
    end += k < a.axes ? a.section[k] : 0;
  }
  return x;
}

// v_rsq_f32 (1 ulp); it takes numbers below the least normal one for zeros.
MIA_DEV float inverse_root(float x) {
  return x < 1e-30f ? 1.0f / sqrtf(x) : __builtin_amdgcn_rsqf(x);
}

constexpr int kMaxRows = 4;  // head rows per lane group at most

// Workgroup (token t, head range): L lanes of 8 channels per head row (head
// dim <= 8 L); the G lane groups take rows g, g + G, ....
// Eight waves per SIMD (64 registers): 2047 tokens of 64 heads with norms 16.2 us, 17.4
// with the seven that 68 leave; quantised rows with norms would spill.
template <int L, int KIND, bool NORM>
__global__ __launch_bounds__(256, KIND <= kBf16 || !NORM ? 8 : 6) void rope_append_kernel(mia_rope_append_args a, int rows) {
  constexpr int G = 256 / L;
  __shared__ __attribute__((aligned(16))) float cs[2][8 * L / 2];
  const int64_t t = blockIdx.x;
  const int grp = threadIdx.x / L, j = threadIdx.x % L;
  const int Hq = a.num_q_heads, Hkv = a.num_kv_heads, d = a.head_dim, R = a.rot_dim;
  const int NH = Hq + (KIND == kRows && !a.v ? Hkv : 2 * Hkv);
  const bool act = 8 * j < d, rot = 8 * j < R;
  // a lane's channels: e0 .. e0 + 3 and e1 .. e1 + 3; in the half split the
  // rotated ones are pairs (e0 + i, e1 + i)
  const bool split = rot && !a.interleaved;
  const int e0 = split ? 4 * j : 8 * j, e1 = split ? R / 2 + 4 * j : 8 * j + 4;
  const float inv_d = 1.0f / (float)d;
  const int h0 = blockIdx.y * G * rows + grp;
  auto source = [&](int hh) {
    const uint16_t *p;
    if (hh < Hq) p = (const uint16_t *)a.q + t * a.q_stride[0] + hh * a.q_stride[1];
    else if (hh < Hq + Hkv) p = (const uint16_t *)a.k + t * a.k_stride[0] + (hh - Hq) * a.k_stride[1];
    else p = (const uint16_t *)a.v + t * a.v_stride[0] + (hh - Hq - Hkv) * a.v_stride[1];
    return p;
  };
  // all rows of the group are under way before the first is used
  u32x4_t raw[kMaxRows];
#pragma unroll
  for (int r = 0; r < kMaxRows; ++r) {
    raw[r] = u32x4_t{0u, 0u, 0u, 0u};
    const int hh = h0 + r * G;
    if (r < rows && hh < NH && act) {
      const uint16_t *p = source(hh);
      const u32x2_t x = *reinterpret_cast<const u32x2_t *>(p + e0);
      const u32x2_t y = *reinterpret_cast<const u32x2_t *>(p + e1);
      raw[r] = u32x4_t{x[0], x[1], y[0], y[1]};
    }
  }
  // the lane's norm weights of Q and K (of lanes past the head dim too: their zeros
  // stay zeros and enter the row's maximum)
  const f32x4_t ones = {1.f, 1.f, 1.f, 1.f};
  f32x4_t gq[2] = {ones, ones}, gk[2] = {ones, ones};
  if (NORM && act) {
    auto four = [&](const void *g, int e) {
      if (!g) return f32x4_t{1.f, 1.f, 1.f, 1.f};
      if (a.gamma_bf16) {
        const u32x2_t w = *reinterpret_cast<const u32x2_t *>((const uint16_t *)g + e);
        return f32x4_t{bf16lo(w[0]), bf16hi(w[0]), bf16lo(w[1]), bf16hi(w[1])};
      }
      return *reinterpret_cast<const f32x4_t *>((const float *)g + e);
    };
    gq[0] = four(a.q_gamma, e0), gq[1] = four(a.q_gamma, e1);
    gk[0] = four(a.k_gamma, e0), gk[1] = four(a.k_gamma, e1);
  }
  int64_t slot = -1, blk = 0, off = 0;
  if constexpr (KIND != kRows) {
    slot = load_int(a.slots, a.slot_dtype, t);
    if (slot >= (int64_t)a.num_blocks * a.block_size) slot = -1;
    if (slot >= 0) {
      blk = slot / a.block_size;
      off = slot - blk * a.block_size;
    }
  }
  // The token's angles, once for all heads: pos * inv_freq in turns, in 64
  // bits (a position of 2^20 leaves 24 bits less of a 32-bit turn), reduced to
  // half a turn, which 32 bits hold to 2^-25.
  for (int i = threadIdx.x; i < R / 2; i += 256) {
    const double pos = (double)load_int(
        a.positions, a.pos_dtype, axis_of(a, i) * a.pos_stride[0] + t * a.pos_stride[1]);
    const double turns = pos * ((double)a.inv_freq[i] * 0.15915494309189533577);
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[0][i] = c * a.rope_scale;
    cs[1][i] = s * a.rope_scale;
  }
  __syncthreads();
  f32x4_t co = {1.f, 1.f, 1.f, 1.f}, si = {0.f, 0.f, 0.f, 0.f};
  if (rot) {
    co = *reinterpret_cast<const f32x4_t *>(&cs[0][4 * j]);
    si = *reinterpret_cast<const f32x4_t *>(&cs[1][4 * j]);
  }
  auto do_row = [&](int hh, const u32x4_t &w) {
    const int kind = hh < Hq ? 0 : hh < Hq + Hkv ? 1 : 2;  // Q, K, V
    const int h = hh - (kind == 0 ? 0 : kind == 1 ? Hq : Hq + Hkv);
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16lo(w[i]);
      x[2 * i + 1] = bf16hi(w[i]);
    }
    if constexpr (NORM) {  // (every lane takes part in the sum)
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int m = L / 2; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
      if (kind != 2) {
        const float rinv = inverse_root(ss * inv_d + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] *= rinv * (kind == 0 ? gq[i >> 2][i & 3] : gk[i >> 2][i & 3]);
      }
    }
    if (kind != 2 && rot) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float &xa = a.interleaved ? x[2 * i] : x[i];
        float &xb = a.interleaved ? x[2 * i + 1] : x[4 + i];
        const float ya = xa * co[i] - xb * si[i];
        xb = xb * co[i] + xa * si[i];
        xa = ya;
      }
    }
    // rounded to bf16 once, behind norm and rotation; codes are of the
    // unrounded values
    const u32x4_t bw = kind == 2 ? w
                                 : u32x4_t{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]),
                                           pack2_bf16(x[4], x[5]), pack2_bf16(x[6], x[7])};
    auto store16 = [&](uint16_t *p) {
      if (!act) return;
      *reinterpret_cast<u32x2_t *>(p + e0) = u32x2_t{bw[0], bw[1]};
      *reinterpret_cast<u32x2_t *>(p + e1) = u32x2_t{bw[2], bw[3]};
    };
    if (kind == 0) {
      store16((uint16_t *)a.q_out + t * a.q_out_stride[0] + h * a.q_out_stride[1]);
      return;
    }
    if (kind == 1 && a.k_out)
      store16((uint16_t *)a.k_out + t * a.k_out_stride[0] + h * a.k_out_stride[1]);
    if constexpr (KIND != kRows) {
      const int64_t *st = kind == 1 ? a.k_cache_stride : a.v_cache_stride;
      const int64_t at = blk * st[0] + h * st[1] + off * st[2];
      uint8_t *pool = (uint8_t *)(kind == 1 ? a.k_cache : a.v_cache);
      if constexpr (KIND == kBf16) {
        if (slot >= 0) store16((uint16_t *)pool + at);
      } else if constexpr (KIND == kFp8Static) {
        if (slot < 0 || !act) return;
        const float *dq = kind == 1 ? a.k_dequant : a.v_dequant;
        const float s = dq ? dq[h] : 1.0f;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = x[i] / s;
          // (keeps NaN, which fminf and fmaxf would drop)
          if (y[i] > 448.0f) y[i] = 448.0f;
          if (y[i] < -448.0f) y[i] = -448.0f;
        }
        *reinterpret_cast<uint32_t *>(pool + at + e0) = e4m3fn_x4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<uint32_t *>(pool + at + e1) = e4m3fn_x4(y[4], y[5], y[6], y[7]);
      } else {
        constexpr int Q = KIND == kI8 ? 127 : 448;
        uint32_t mag = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mag = max(mag, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
        for (int m = L / 2; m >= 1; m >>= 1) mag = max(mag, (uint32_t)__shfl_xor((int)mag, m, 64));
        if (slot < 0 || !act) return;
        RowCodes<Q> rc;
        rc.set(mag);
        uint32_t c4[2] = {0u, 0u};
        if constexpr (KIND == kI8) {
#pragma unroll
          for (int i = 0; i < 8; ++i) c4[i >> 2] |= rc.int8(x[i]) << (8 * (i & 3));
        } else {
          c4[0] = e4m3fn_x4(rc.code(x[0]), rc.code(x[1]), rc.code(x[2]), rc.code(x[3]));
          c4[1] = e4m3fn_x4(rc.code(x[4]), rc.code(x[5]), rc.code(x[6]), rc.code(x[7]));
        }
        *reinterpret_cast<uint32_t *>(pool + at + e0) = c4[0];
        *reinterpret_cast<uint32_t *>(pool + at + e1) = c4[1];
        if (j == 0) {
          const int64_t *ss = kind == 1 ? a.k_scale_stride : a.v_scale_stride;
          float *sc = kind == 1 ? a.k_scales : a.v_scales;
          sc[blk * ss[0] + h * ss[1] + off * ss[2]] = cache_scale<Q>(mag);
        }
      }
    }
  };
  // one copy of the row code (the rows shift down the loaded registers)
#pragma nounroll
  for (int r = 0; r < rows; ++r) {
    const int hh = h0 + r * G;
    if (hh >= NH) break;
    do_row(hh, raw[0]);
#pragma unroll
    for (int m = 0; m + 1 < kMaxRows; ++m) raw[m] = raw[m + 1];
  }
}

template <int L, bool NORM>
void launch_lanes(const mia_rope_append_args &a, int kind, hipStream_t s) {
  constexpr int G = 256 / L;
  const int heads = a.num_q_heads + (a.v ? 2 : 1) * a.num_kv_heads;
  const int sets = (heads + G - 1) / G;  // rows per group in one workgroup per token
  // Few tokens need workgroups, many of them fewer repeated angles and loads in
  // flight: rows of 1 / 2 / 3 / 4 per group, 64 heads of d = 128 with norms, 100
  // tokens 4.4 / 4.8 / 4.8 / 6.0 us, 512 7.7 / 7.6 / 7.7 / 8.1, 2047 20.3 / 17.8 / 17.5
  // / 16.4; 48 heads, 16383 tokens 98 / 91 / 78 / 76.
  const int most = a.num_tokens < 256 ? 1 : a.num_tokens < 1024 ? 2 : kMaxRows;
  const int parts = (sets + most - 1) / most;
  const int rows = (sets + parts - 1) / parts;
  const dim3 grid((unsigned)a.num_tokens, (sets + rows - 1) / rows);
  switch (kind) {
    case kRows: rope_append_kernel<L, kRows, NORM><<<grid, 256, 0, s>>>(a, rows); break;
    case kBf16: rope_append_kernel<L, kBf16, NORM><<<grid, 256, 0, s>>>(a, rows); break;
    case kFp8Static: rope_append_kernel<L, kFp8Static, NORM><<<grid, 256, 0, s>>>(a, rows); break;
    case kFp8: rope_append_kernel<L, kFp8, NORM><<<grid, 256, 0, s>>>(a, rows); break;
    default: rope_append_kernel<L, kI8, NORM><<<grid, 256, 0, s>>>(a, rows);
  }
}

template <bool NORM>
void launch_norm(const mia_rope_append_args &a, int kind, hipStream_t s) {
  if (a.head_dim <= 64) launch_lanes<8, NORM>(a, kind, s);
  else if (a.head_dim <= 128) launch_lanes<16, NORM>(a, kind, s);
  else launch_lanes<32, NORM>(a, kind, s);
}

}  // namespace

int launch_rope_append(const mia_rope_append_args &a, hipStream_t s) {
  const int kind = !a.slots ? kRows
                   : a.cache_dtype == MIA_DTYPE_BF16 ? kBf16
                   : a.cache_dtype == MIA_DTYPE_I8 ? kI8
                   : a.k_scales ? kFp8 : kFp8Static;
  if (a.qk_norm) launch_norm<true>(a, kind, s);
  else launch_norm<false>(a, kind, s);
  return check_hip(hipGetLastError(), "rope_kv_append");
}

}  // namespace mia
