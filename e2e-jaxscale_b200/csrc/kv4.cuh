// Pages of the 4-bit key/value cache (kv4.cu, kv4_attn.cu).
//
// A pool is [num_pages][nkv][block]; the block of one page and one kv head holds
// page_tokens rows of K and of V:
//   K codes [pt][D / 2] | V codes [pt][D / 2] | K scales [pt][D / 16] | V scales [pt][D / 16]
// with two e2m1 codes per byte (even dimension in the low half) and one e4m3
// scale per 16 values of a row: 4.5 bits per value.  A stored value is
// code x scale.  Codes have 2 significant bits and scales 4, so the product has
// at most 6 and lies in [2^-10, 2688]: it is exact in f16 and in bf16, and no
// reader rounds.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace jsx {

constexpr int kKv4Group = 16;  // values per scale

// bytes of one page's block for one kv head
__host__ __device__ constexpr int kv4_block_bytes(int pt, int D) { return pt * D + pt * (D / 8); }
__host__ __device__ constexpr int kv4_off_v(int pt, int D) { return pt * (D / 2); }
__host__ __device__ constexpr int kv4_off_ks(int pt, int D) { return pt * D; }
__host__ __device__ constexpr int kv4_off_vs(int pt, int D) { return pt * D + pt * (D / 16); }

inline bool kv4_page_tokens_ok(int pt) { return pt == 16 || pt == 32 || pt == 64 || pt == 128; }

// host checks shared by the entry points that take a pool and a page table
#define JSX_KV4_REQUIRE(pool, num_pages, table, table_slots, nkv, head_dim, page_tokens)                        \
  do {                                                                                                          \
    JSX_REQUIRE((pool) && (table), "null pool or page table");                                                  \
    JSX_REQUIRE(::jsx::aligned16(pool) && ::jsx::aligned4(table), "pool must be 16-byte aligned, the table 4"); \
    JSX_REQUIRE((num_pages) >= 1 && (table_slots) >= 1 && (nkv) >= 1, "num_pages=%d table_slots=%d nkv=%d",      \
                (int)(num_pages), (int)(table_slots), (int)(nkv));                                              \
    JSX_REQUIRE(::jsx::kv4_page_tokens_ok(page_tokens), "page_tokens=%d is not 16, 32, 64 or 128",               \
                (int)(page_tokens));                                                                            \
    if ((head_dim) != 64 && (head_dim) != 128) {                                                                \
      ::jsx::set_error("head_dim=%d (the 4-bit cache takes 64 and 128)", (int)(head_dim));                       \
      return JSX_ENOTSUP;                                                                                       \
    }                                                                                                           \
  } while (0)

// the four bytes of a word -> four f16x2.  The word has to be a whole 32-bit load:
// nvcc 12.9 turns the conversion of a zero-extended byte load into zeros.
__device__ __forceinline__ void e2m1x8_to_h2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n"
      " cvt.rn.f16x2.e2m1x2 %1, b;\n cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// two e4m3 scales (low byte first) -> f16x2
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t two) {
  uint32_t r;
  asm("{\n .reg .b16 a;\n cvt.u16.u32 a, %1;\n cvt.rn.f16x2.e4m3x2 %0, a;\n}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t hmul2_u(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// eight f32 -> eight e2m1 codes (the first in the low bits), round to nearest even, saturating
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float (&x)[8]) {
  uint32_t r;
  asm("{\n .reg .b8 a, b, c, d;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return r;
}
// f32 -> e4m3 (round to nearest even, saturating at 448, NaN stays NaN) and its value
__device__ __forceinline__ uint32_t f32_to_e4m3(float x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
  return (uint32_t)r & 0xffu;
}

}  // namespace jsx
