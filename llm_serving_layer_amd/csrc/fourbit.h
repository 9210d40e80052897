// The 4-bit cache's format: what a page holds and where.
//
// A row of a KV head (one token's K or V) is cut into groups of 64 elements, or
// is one group where head_dim is no multiple of 64. A group keeps
//   zero  the largest float16 that is not above its least element,
//   step  the least float16 that is not below (largest - zero) / 15,
//   c     per element, (x - zero) / step rounded to the nearest whole number
//         (ties to even), at most 15,
// and stands for zero + c step. Elements beyond +-65504 are brought to that
// first; a group with a NaN or an infinity gets NaN for both and reads as NaN.
// The zero is not above and 15 steps reach the largest element, so a value
// stands half a step from its element at most.
//
// A block's K (or V) is n_kv_heads heads of page_size x head_dim / 2 bytes of
// codes, then (16-byte aligned) [head][group][row] words, the step in the upper
// half and the zero in the lower. Rows of 16 make a tile where page_size and
// head_dim are multiples of 16 and 64 ("tiled"), laid out for the matrix cores'
// operands (lane 16 g + n):
//   K  row after row; in a row, 16-element block 4 q + g (group q) at bytes
//      8 (g groups + q): a lane's blocks of all groups lie together;
//   V  byte (16 g + n) head_dim / 8 + 4 b + j holds dims 32 b + n (low half) and
//      32 b + 16 + n (high) of row 4 g + j: a lane's four rows are one word,
//      and a byte belongs to one row, so rows are written independently.
// A byte of K holds elements 2 i (low) and 2 i + 1. Elsewhere K and V are row
// after row, a byte two elements.
#pragma once

#include "mfma.h"

namespace pkv {

struct FourBit {
  int32_t n_kv, d, ps, groups;
  bool tiled;
  int32_t head_bytes;    // codes of a head
  int32_t pairs;         // where a block's words begin
  int64_t block;         // bytes of a block's K (or V)
};

__host__ __device__ inline FourBit four_bit(int32_t n_kv, int32_t d, int32_t ps) {
  FourBit f;
  f.n_kv = n_kv;
  f.d = d;
  f.ps = ps;
  f.groups = d % 64 == 0 ? d / 64 : 1;
  f.tiled = d % 64 == 0 && ps % 16 == 0;
  f.head_bytes = ps * (d / 2);
  f.pairs = (n_kv * f.head_bytes + 15) / 16 * 16;
  f.block = ((int64_t)f.pairs + (int64_t)n_kv * f.groups * ps * 4 + 15) / 16 * 16;
  return f;
}

// n / d for n < 2^31 as a product: with 2^s >= d and m = 2^(31 + s) / d rounded up (by
// less than 2^s / d), n m exceeds n 2^(31 + s) / d by less than 2^(31 + s) / d.
struct Div {
  uint32_t d, m;
  int32_t s;
};
inline Div div_by(uint32_t d) {
  int s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Div& v, uint32_t& rest) {
  const uint32_t q = (uint32_t)((uint64_t)n * v.m >> v.s);
  rest = n - q * v.d;
  return q;
}

// Where row r's element e lies among a head's codes: byte and half.
__device__ __forceinline__ int k_byte(const FourBit& f, int r, int e) {
  if (!f.tiled) return r * (f.d / 2) + e / 2;
  const int q = e >> 6, g = (e >> 4) & 3;
  return r * (f.d / 2) + (g * f.groups + q) * 8 + (e & 15) / 2;
}
__device__ __forceinline__ int k_half(const FourBit&, int e) { return e & 1; }
__device__ __forceinline__ int v_byte(const FourBit& f, int r, int e) {
  if (!f.tiled) return r * (f.d / 2) + e / 2;
  const int row = r & 15;
  return (r >> 4) * 8 * f.d + ((row >> 2) * 16 + (e & 15)) * (f.d / 8) + (e >> 5) * 4 + (row & 3);
}
__device__ __forceinline__ int v_half(const FourBit& f, int e) {
  return f.tiled ? (e >> 4) & 1 : e & 1;
}
__device__ __forceinline__ int group_of(const FourBit& f, int e) {
  return f.groups == 1 ? 0 : e >> 6;
}

// The word's two halves. (Built from the integers, so a NaN keeps its bits.)
__device__ __forceinline__ _Float16 f16_bits(uint32_t b) {
  return __builtin_bit_cast(_Float16, (uint16_t)b);
}
__device__ __forceinline__ float pair_step(uint32_t w) { return (float)f16_bits(w >> 16); }
__device__ __forceinline__ float pair_zero(uint32_t w) { return (float)f16_bits(w & 0xffffu); }

// The float16 below (above) h, for finite h.
__device__ __forceinline__ _Float16 next_f16(_Float16 h, bool up) {
  const int16_t b = __builtin_bit_cast(int16_t, h);
  if ((b & 0x7fff) == 0) return f16_bits(up ? 0x0001u : 0x8001u);
  return f16_bits((uint32_t)((b > 0) == up ? b + 1 : b - 1));
}

constexpr float kF16Max = 65504.f;
constexpr uint32_t kNanPair = 0x7e007e00u;

// A group's word, from its least and largest element (finite, in range). The nearest
// float16 to the quotient (in 32 bits: off by 2^-22 of it) is the step or the one
// below it: 15 steps, exact in 32 bits, against the difference in 64 decide.
__device__ __forceinline__ uint32_t group_pair(float lo, float hi) {
  _Float16 z = (_Float16)lo;
  if ((float)z > lo) z = next_f16(z, false);
  const double need = (double)hi - (double)(float)z;
  uint32_t s = __builtin_bit_cast(uint16_t, (_Float16)((float)need * (1.f / 15.f)));
  s += (double)(15.f * (float)f16_bits(s)) < need;
  return s << 16 | __builtin_bit_cast(uint16_t, z);
}

// Element x's code. In 32 bits with an error below 2^-17 steps; next to a
// border (closer than 2^-14) the order against it is decided in 64 bits.
__device__ __forceinline__ uint32_t code_of(float x, float step, float inv, float zero) {
  const float t = (x - zero) * inv;
  float k = __builtin_floorf(t);
  const float past = t - k - 0.5f;
  if (__builtin_fabsf(past) < 0x1p-14f) {
    const double twice = 2.0 * ((double)x - (double)zero);
    const double border = (2.0 * (double)k + 1.0) * (double)step;
    if (twice > border || (twice == border && ((int)k & 1))) k += 1.f;
  } else if (past > 0.f) {
    k += 1.f;
  }
  k = step > 0.f ? fminf(k, 15.f) : 0.f;
  return (uint32_t)(int)k;
}

}  // namespace pkv
