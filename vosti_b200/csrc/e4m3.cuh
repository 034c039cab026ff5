// A paged cache of 8 bits: float8 e4m3 payloads with a power of two for every block of 16 tokens and kv head, keys and
// values apart. What is held is payload * 2^(scale - 127); a scale of 255 is no number, and neither is what its block holds.
//   keys      [pages, kv heads, page, d]               a token's key is d bytes side by side
//   values    [pages, kv heads, page / 16, d, 16]      inside a block a feature's 16 values lie side by side
//   scales    [pages, kv heads, page / 16]             one byte each, keys and values
// Feature-major values are what a matrix instruction wants of the weights' product (its k index, the token, runs along a
// lane's word); the writer turns a block once, readers would have to turn it at every step.
// (One is also where a size of 2^96 or more was to be held.) The payloads 0x7f and 0xff are no numbers either; a store leaves them in such blocks only.
// A power of two as the scale costs e4m3 nothing (its own exponent moves), makes what is held exact in bfloat16, and lets a
// block take a larger scale by moving exponents: only values that fall below e4m3's 2^-6 are rounded a second time.
#pragma once
#include "common.cuh"

constexpr int E4M3_BLOCK = 16;             // tokens of a block with one scale
constexpr int E4M3_NAN_SCALE = 255;
// Sizes from here on count as no numbers. Attention sums weights of up to 2^8 (a running maximum that follows lazily) times values
// before it divides: 2^8 * 2^23 keys * 2^96 is still below float32's 2^128.
constexpr float E4M3_LIMIT = 79228162514264337593543950336.f;   // 2^96

// Two floats as payloads, ties to even, at most 448 in size; `lo` in the low byte.
__device__ __forceinline__ uint16_t e4m3_pack(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two payloads as floats.
__device__ __forceinline__ float2 e4m3_unpack(uint16_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
  float2 r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(r.x), "=f"(r.y) : "r"(h));
  return r;
}
// 2^(scale - 127), not a number for 255.
__host__ __device__ __forceinline__ float e4m3_scale(int scale) {
  union { uint32_t u; float f; } v;
  v.u = scale == E4M3_NAN_SCALE ? 0x7fffffffu : scale == 0 ? 0x00400000u : (uint32_t)scale << 23;
  return v.f;
}
// The smallest scale that brings a largest size of `amax` (finite, >= 0) to 448 = 1.75 * 2^8 or below.
__device__ __forceinline__ int e4m3_scale_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int scale = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return scale > 0 ? scale : 0;
}

// ---- payloads as bfloat16: bits in their new places, and a product with a power of two for the difference of the exponents' biases, which takes
// subnormals with it (published for float16 by F. Giesen, "Half to float done quick", 2012)
__device__ __forceinline__ uint32_t bf16x2_times(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A payload's bits moved into bfloat16's places stand for its value times 2^-120 (the formats' exponents are biased by 7 and 127), its
// subnormals included (0x7f and 0xff come out as 480 and have to be looked for). The block's factor is 2^120 * 2^(scale - 127); what of it is above bfloat16's range is a second one.
struct E4m3Factor { uint32_t first, second; };
constexpr uint32_t E4M3_ONE = 0x3f803f80u;
__device__ __forceinline__ E4m3Factor e4m3_factor(int scale) {
  if (scale == E4M3_NAN_SCALE) return {0x7fff7fffu, E4M3_ONE};
  const int e = scale - 7, lo = e < 127 ? e : 127;             // e: -7 .. 247
  return {(uint32_t)((lo + 127) << 7) * 0x10001u, (uint32_t)((e - lo + 127) << 7) * 0x10001u};
}
// Payload bytes 2 I and 2 I + 1 of a word, times the first factor (each byte with copies of its sign above it, moved up: sign, zeros, exponent, mantissa).
template <int I>
__device__ __forceinline__ uint32_t e4m3_widen(uint32_t w, const E4m3Factor& f) {
  uint32_t x;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(x) : "r"(w), "n"(I == 0 ? 0x9180 : 0xb3a2));
  return bf16x2_times((x << 4) & 0x87f087f0u, f.first);
}
// Bit 7 of every byte of a word that is no number's payload, and other bits of no meaning.
constexpr uint32_t E4M3_NO_NUMBERS = 0x80808080u;
__device__ __forceinline__ uint32_t e4m3_no_numbers(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u; }
// A mask of the first n bytes of a word (n <= 0: none, n >= 4: all).
__device__ __forceinline__ uint32_t e4m3_first_bytes(int n) { return n <= 0 ? 0u : n >= 4 ? 0xffffffffu : (1u << (8 * n)) - 1u; }
