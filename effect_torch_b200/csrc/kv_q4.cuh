// The 4-bit KV tier: rows cut into blocks of 32 values with an f16 scale, by the Q4_0 rule (quant_kernels.cu): the value of largest
// magnitude divided by -8 is the scale d, a code is floor(x / d + 8.5) held to 0..15 and stands for (code - 8) * d.
//
// One record per (page, KV head): the codes of its rows, head_dim / 2 bytes each, then their scales, head_dim / 32 f16 each; 18
// bytes per block as in a GGUF row, and one contiguous run per page and head (1152 bytes for 16 rows of 128). Codes lie in a row so that
// a thread of an m16n8k16 product finds its operands side by side (attention_q4.cu). With nb = head_dim / 32 blocks b:
//   K: words [t][b], t < 4: elements 8 t .. 8 t + 7 of the block; even ones in the low half, odd ones in the high half, ascending
//   V: half words [g][b], g < 8: elements g, g + 8, g + 16, g + 24 of the block, ascending; those of two neighbouring rows alternate (pages
//      of an odd number of rows: row by row)
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "kernels.h"

namespace etc {

__host__ __device__ __forceinline__ size_t q4_record_bytes(int block_size, int head_dim) { return (size_t)block_size * (head_dim / 32) * 18; }

// Where a row's codes begin and how far apart its half words are.
struct Q4Row {
  uint16_t* codes;
  __half* scales;
  int stride;
};
__device__ __forceinline__ Q4Row q4_row(const PoolView& p, bool is_v, int page, int head, int slot) {
  uint8_t* record = reinterpret_cast<uint8_t*>(is_v ? p.v : p.k) + ((size_t)page * p.kv_heads + head) * q4_record_bytes(p.block_size, p.head_dim);
  const int row_halves = p.head_dim / 4;
  const bool paired = is_v && p.block_size % 2 == 0;
  uint16_t* codes = reinterpret_cast<uint16_t*>(record);
  return {paired ? codes + (size_t)(slot & ~1) * row_halves + (slot & 1) : codes + (size_t)slot * row_halves,
          reinterpret_cast<__half*>(codes + (size_t)p.block_size * row_halves) + (size_t)slot * (p.head_dim / 32), paired ? 2 : 1};
}

// One element, for the paths that are not in a hurry.
__device__ __forceinline__ float q4_value(const Q4Row& row, bool is_v, int d, int nb) {
  const int b = d >> 5, e = d & 31;
  const int half = is_v ? ((e & 7) * nb + b) * row.stride : 2 * ((e >> 3) * nb + b) + (e & 1), shift = is_v ? (e >> 3) * 4 : ((e & 7) >> 1) * 4;
  return __fmul_rn((float)(((row.codes[half] >> shift) & 15) - 8), __half2float(row.scales[b]));
}

// Quantizes a block by four neighbouring lanes, lane t of which (the lowest two bits) holds elements 8 t .. 8 t + 7, and stores it where
// `live`. All lanes of the warp take part; the four of a block agree on everything but the values.
__device__ __forceinline__ void q4_store_block(const float (&v)[8], bool is_v, const Q4Row& row, int b, int nb, bool live) {
  const int t = threadIdx.x & 3;
  float extreme = 0.0f;  // a NaN is never taken
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (fabsf(v[i]) > fabsf(extreme)) extreme = v[i];
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, extreme, off);
    if (fabsf(o) > fabsf(extreme) || (fabsf(o) == fabsf(extreme) && (t & off))) extreme = o;  // of equals the first
  }
  const float d = __fmul_rn(extreme, -0.125f), inv = d != 0.0f ? __frcp_rn(d) : 0.0f;
  // The floor of a value in [0, 16) is the low byte of it plus 2^23, rounded down. Codes are shifted and added with the exponent that the
  // sums have; what the exponents come to is taken off at the end.
  auto pack = [&](auto shift_of) {
    constexpr uint32_t kExponent = 0x4B000000u;
    uint32_t word = 0, extra = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      word += __float_as_uint(__fadd_rd(fminf(fmaxf(__fadd_rn(__fmul_rn(v[i], inv), 8.5f), 0.0f), 15.5f), 8388608.0f)) << shift_of(i);
      extra += kExponent << shift_of(i);
    }
    return word - extra;
  };
  if (is_v) {
    // element 8 t + g is code t of half word g: byte s of a lane's word holds its codes for g = 2 s and 2 s + 1
    const uint32_t mine = pack([](int i) { return 4 * i; });
    uint32_t w[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) w[s] = __shfl_sync(0xffffffffu, mine, s, 4);
    const unsigned pick = (unsigned)(t | (t + 4) << 4);
    const uint32_t bytes = __byte_perm(__byte_perm(w[0], w[1], pick), __byte_perm(w[2], w[3], pick), 0x5410);
    auto nibbles = [](uint32_t x) {  // the low ones of the four bytes, side by side
      x &= 0x0F0F0F0Fu;
      x |= x >> 4;
      return __byte_perm(x, 0u, 0x4420) & 0xFFFFu;
    };
    const uint32_t even = nibbles(bytes), odd = nibbles(bytes >> 4);
    if (live) {
      row.codes[(2 * t * nb + b) * row.stride] = (uint16_t)even;
      row.codes[((2 * t + 1) * nb + b) * row.stride] = (uint16_t)odd;
    }
  } else if (live) {
    const uint32_t word = pack([](int i) { return 4 * (i >> 1) + 16 * (i & 1); });
    uint16_t* dst = row.codes + 2 * (t * nb + b);
    if ((reinterpret_cast<uintptr_t>(dst) & 3) == 0) {
      *reinterpret_cast<uint32_t*>(dst) = word;
    } else {  // pages of an odd number of blocks
      dst[0] = (uint16_t)word;
      dst[1] = (uint16_t)(word >> 16);
    }
  }
  if (live && t == 0) row.scales[b] = __float2half_rn(d);
}

// The reverse in two halves: what a lane fetches of block b, and elements 8 t .. 8 t + 7 of it.
struct Q4Part {
  uint32_t word;
  float scale;
};
__device__ __forceinline__ Q4Part q4_fetch(const Q4Row& row, bool is_v, int b, int nb) {
  const int t = threadIdx.x & 3;
  const int at = is_v ? (2 * t * nb + b) * row.stride : 2 * (t * nb + b), next = is_v ? at + nb * row.stride : at + 1;
  return {row.codes[at] | (uint32_t)row.codes[next] << 16, __half2float(row.scales[b])};
}
__device__ __forceinline__ void q4_unpack(const Q4Part& part, bool is_v, float (&v)[8]) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t code;
    if (is_v) code = __shfl_sync(0xffffffffu, part.word, i >> 1, 4) >> (4 * t + 16 * (i & 1));
    else code = part.word >> (4 * (i >> 1) + 16 * (i & 1));
    // 2^23 + code less 2^23 + 8: a conversion from integers would take the slowest pipe
    v[i] = __fmul_rn(__fsub_rn(__uint_as_float((code & 15u) | 0x4B000000u), 8388616.0f), part.scale);
  }
}

}  // namespace etc
