// The 4-bit KV cache's page layout and its dequantisation, shared by the kernels that write it, read it
// back and attend over it.
//
// A value is bf16(s c + b): codes c in 0..15, bf16 scale s and bias b per 64 dims, in the 8-bit cache's
// words (s | b << 16) [page][kv head][token][hd/64]. The codes of a page of one kv head take
// page * hd / 2 bytes and lie as the matrix instructions of the attention kernels take them, so that a
// wave's 16-byte loads are whole operands (lane l of 64: n = l % 16, g = l / 16):
//   K  one row of hd / 2 bytes per token. The A operand of S^T = K . Q^T holds key n, dims 32 s + 8 g ..
//      + 7 for step s: word s % 4 of the lane's 16 bytes at 64 (s / 4) + 16 g, dim 8 g + e its half byte e.
//   V  blocks of 32 tokens, 16 hd bytes each. The A operand of O^T = V^T . P^T holds dim n of a 16-dim
//      tile and 8 keys: those whose probabilities the same lane holds after S^T, keys 4 g + r and
//      16 + 4 g + r. Chunk c (64 dims): the lane's 16 bytes at 1024 c + 16 l, byte 8 p + 4 u + r = key
//      16 u + 4 g + r, dim 64 c + 32 p + n in its low half and 16 dims on in its high half.
// A token's K and V rows are whole bytes, so tokens are written apart from each other.
#pragma once

#include "common.h"

namespace dsk {

constexpr int kKv4Block = 32;  // tokens per V block: pages are multiples of it

// byte offset, within its token's K row, of the word that holds dims 8 sub .. 8 sub + 7
__host__ __device__ __forceinline__ int kv4_k_word(int sub) { return (sub / 16) * 64 + (sub % 4) * 16 + (sub % 16) / 4 * 4; }

// byte offset, within its page, of token t, dim d of V (the low half byte: d % 32 < 16)
__host__ __device__ __forceinline__ int kv4_v_byte(int hd, int t, int d) {
  return (t / 32) * 16 * hd + (d / 64) * 1024 + ((d % 16) + 16 * ((t % 16) / 4)) * 16 + ((d % 64) / 32) * 8 +
         ((t % 32) / 16) * 4 + t % 4;
}

// A half byte in place in a word is the float16 denormal c 2^-24 (bits 0..3 of a half) or c 2^-20 (bits
// 4..7): v_fma_mix_f32 takes it as it is, so 8 codes cost 5 masks and shifts, 8 fmas and 4 packs. The
// scale arrives times 2^24 and 2^20, by adding to its exponent: exact for s in [2^-126, 2^103), which
// leaves values up to 1e31 (a smaller scale reads back within 1e-37 of its values).
struct Kv4Scale {
  float s24, s20, b;
};
__device__ __forceinline__ Kv4Scale kv4_scale(uint32_t w) {
  uint32_t s24;  // one instruction, which the compiler splits into two to share the shift
  asm("v_lshl_add_u32 %0, %1, 16, %2" : "=v"(s24) : "v"(w), "s"(24u << 23));
  return Kv4Scale{bits_f32(s24), bits_f32(s24 - (4u << 23)), bits_f32(w & 0xffff0000u)};
}

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float kv4_lo(uint32_t m, float s, float b) {
  return __builtin_fmaf((float)__builtin_bit_cast(half2_t, m)[0], s, b);
}
__device__ __forceinline__ float kv4_hi(uint32_t m, float s, float b) {
  return __builtin_fmaf((float)__builtin_bit_cast(half2_t, m)[1], s, b);
}

// 8 half bytes of one scale -> 8 bf16 values, half byte e to element e
__device__ __forceinline__ u32x4 kv4_row8(uint32_t w, const Kv4Scale& z) {
  const uint32_t a = w & 0x000f000fu, b = w & 0x00f000f0u, w8 = w >> 8;
  const uint32_t c = w8 & 0x000f000fu, d = w8 & 0x00f000f0u;
  return u32x4{pack_bf16x2(kv4_lo(a, z.s24, z.b), kv4_lo(b, z.s20, z.b)), pack_bf16x2(kv4_lo(c, z.s24, z.b), kv4_lo(d, z.s20, z.b)),
               pack_bf16x2(kv4_hi(a, z.s24, z.b), kv4_hi(b, z.s20, z.b)), pack_bf16x2(kv4_hi(c, z.s24, z.b), kv4_hi(d, z.s20, z.b))};
}

// A word of V: 4 tokens (scales z) of dim d (low halves) and d + 16 (high halves) -> two bf16 pairs each
__device__ __forceinline__ void kv4_col4(uint32_t w, const Kv4Scale* z, uint32_t (&lo)[2], uint32_t (&hi)[2]) {
  const uint32_t a = w & 0x000f000fu, b = w & 0x00f000f0u, w8 = w >> 8;
  const uint32_t c = w8 & 0x000f000fu, d = w8 & 0x00f000f0u;
  lo[0] = pack_bf16x2(kv4_lo(a, z[0].s24, z[0].b), kv4_lo(c, z[1].s24, z[1].b));
  lo[1] = pack_bf16x2(kv4_hi(a, z[2].s24, z[2].b), kv4_hi(c, z[3].s24, z[3].b));
  hi[0] = pack_bf16x2(kv4_lo(b, z[0].s20, z[0].b), kv4_lo(d, z[1].s20, z[1].b));
  hi[1] = pack_bf16x2(kv4_hi(b, z[2].s20, z[2].b), kv4_hi(d, z[3].s20, z[3].b));
}

}  // namespace dsk
