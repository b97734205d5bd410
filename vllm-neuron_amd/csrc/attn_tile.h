// attn_tile.h — device pieces shared by the attention kernels that walk key
// tiles of paged caches: cache kinds and their widening to bf16, LDS swizzles
// and copies, lane reductions, and the joining of partial results.
#pragma once

#include "mia_device.h"
#include "mia_internal.h"

namespace mia {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
typedef __attribute__((address_space(3))) uint8_t lds_u8_t;
typedef __attribute__((address_space(3))) u32x2_t lds_u32x2_t;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4_t;
typedef __attribute__((address_space(3))) f32x4_t lds_f32x4_t;
typedef __attribute__((address_space(3))) float lds_f32_t;

enum CacheKind { kBf16 = 0, kFp8 = 1, kI8 = 2 };

// Lengths and tables through the scalar cache: nothing writes them while the
// kernel runs, which the compiler cannot know of a plain pointer.
MIA_DEV int scalar_load(const int32_t *p, int64_t i) {
  return ((const __attribute__((address_space(4))) int32_t *)(uintptr_t)p)[i];
}

template <int D>
MIA_DEV constexpr int k_swz(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
MIA_DEV constexpr int v_swz(int row) { return D == 128 ? (row & 3) << 2 : (row & 2) << 1; }

// 8 codes (two dwords) -> 8 bf16 (exact).
template <int CT>
MIA_DEV u32x4_t widen8(uint32_t a, uint32_t b) {
  u32x4_t o;
  if constexpr (CT == kFp8) {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
  } else {
    // (one conversion per value: the byte is picked and extended by the operand)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t u = i ? b : a;
      o[2 * i] = pack2_bf16((float)(int8_t)(u & 0xffu), (float)(int8_t)((u >> 8) & 0xffu));
      o[2 * i + 1] = pack2_bf16((float)(int8_t)((u >> 16) & 0xffu), (float)(int8_t)(u >> 24));
    }
  }
  return o;
}

// over the lanes l and l ^ 32
MIA_DEV float max32(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                   false, false);
  return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}
MIA_DEV float sum32(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                   false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}
// over the lanes l and l ^ 16
MIA_DEV float max16(float x) {
  const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x),
                                                   false, false);
  return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}
MIA_DEV float sum16(float x) {
  const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x),
                                                   false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

// NP 16-byte-per-lane copies HBM -> LDS: lane data of copy j, from src +
// off[j], lands at lds_dst + j * 1024 + 16 * lane; inactive lanes leave theirs.
// Inline assembly, so that the compiler adds no waits before reads of the
// other stage; the wait for the copies is explicit.  M0 (the LDS base of a
// copy) is saved and restored around them.
template <int NP>
MIA_DEV void copy16(const uint8_t *src, const uint32_t (&off)[NP], uint32_t lds_dst) {
  static_assert(NP == 2 || NP == 4, "copies per tile");
  const uint32_t m0 = readfirstlane((int)lds_dst);
  uint32_t saved;
  if constexpr (NP == 4) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %2\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %4, %2\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %5, %2\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %6, %2\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(m0), "s"(src), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3])
        : "memory", "scc");
  } else {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %3, %2\n\t"
        "s_add_u32 m0, m0, 0x400\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %4, %2\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(m0), "s"(src), "v"(off[0]), "v"(off[1])
        : "memory", "scc");
  }
}

// One such copy.
MIA_DEV void copy1(const uint8_t *src, uint32_t off, uint32_t lds_dst) {
  const uint32_t m0 = readfirstlane((int)lds_dst);
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %3, %2\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(m0), "s"(src), "v"(off)
      : "memory");
}

MIA_DEV void add_piece(float &m, float &l, f32x4_t &o, float m1, float l1, const f32x4_t &o1) {
  const float m2 = fmaxf(m, m1);
  const float mm = m2 == -INFINITY ? 0.f : m2;
  const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mm);
  const float b = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - mm);
  m = m2;
  l = l * a + l1 * b;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = o[i] * a + o1[i] * b;
}

// Compute units of the current device.
int cu_count() {
  static int cache[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cache[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        n <= 0)
      n = 256;
    cache[dev] = n;
  }
  return cache[dev];
}

}  // namespace
}  // namespace mia
