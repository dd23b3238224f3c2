// The numbers and the layout of a 4-bit cache.
//
// A number is a sign bit, two exponent bits and a mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; 32 neighbouring channels of a
// token's head share a power of two 2^e, kept as the byte e + 127 (1 .. 254): 17/32 byte a channel. gfx950 turns a byte of two codes and
// its scale into two bfloat16 in one instruction, exactly.
//
// A pool is [pages, heads, bytes]; a page's head is tiles of 16 tokens, so laid out that a lane of the matrix instructions 16 x 16 x 32 finds
// what it needs in one load (attention_4bit.hip):
//   keys:   codes [16 tokens][D / 2], scales [16 tokens][D / 32]: a lane (token, quarter of the channels) reads D / 8 bytes;
//   values: codes [4 quads of tokens][16 lanes][4 tokens][D / 32 bytes], scales [D / 32][16 tokens]: a lane has D / 16 channels and reads
//           four tokens of them.
// Two channels share a byte, the lower one in its lower half.
#pragma once

#include "serving_common.h"

namespace cai {
namespace serving {

constexpr int TILE = 16;   // tokens of a tile

template <int D>
struct Tile4 {
  static constexpr int CODES = TILE * D / 2, BYTES = CODES + TILE * D / 32;
  // of a token's row of keys, and of its 8 channels from c0 on (a multiple of 8) of values
  static DEV_INLINE int key_codes(int t) { return t * (D / 2); }
  static DEV_INLINE int key_scale(int t, int group) { return CODES + t * (D / 32) + group; }
  static DEV_INLINE int value_codes(int t, int c0) {
    return (((t >> 2) * 16 + c0 / (D / 16)) * 4 + (t & 3)) * (D / 32) + (c0 % (D / 16)) / 2;
  }
  static DEV_INLINE int value_scale(int t, int group) { return CODES + group * TILE + t; }
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// two numbers of codes (a byte of `word`) times a power of two
template <int BYTE>
DEV_INLINE unsigned int two_numbers(unsigned int word, float scale) {
  return __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, BYTE));
}
// A scale's byte e + 127 as the conversion takes it: by the exponent's bits, 0 as 2^-127 (measured on gfx950), and with 255 every code, 0 too, becomes
// NaN, so that a key of such a group makes every score NaN whatever the queries' signs (test_cache_4bit_forms.py holds the kernels to it).
DEV_INLINE float scale_of(unsigned int byte) { return __builtin_bit_cast(float, byte << 23); }

// bytes of a page's head
inline int64_t page_bytes(int64_t page_size, int64_t D) { return page_size / TILE * (TILE * D / 2 + TILE * D / 32); }

// The page size of a pool of heads of D channels; 0 if it is no such pool, or does not lie at a 16-byte address.
inline int64_t page_size_of(const at::Tensor& pool, int64_t D) {
  if (pool.dim() != 3 || pool.scalar_type() != at::kByte || !pool.is_contiguous() || reinterpret_cast<uintptr_t>(pool.data_ptr()) % 16 != 0) return 0;
  const int64_t ps = pool.size(2) * 32 / (17 * D);
  return ps >= TILE && (ps & (ps - 1)) == 0 && page_bytes(ps, D) == pool.size(2) ? ps : 0;
}

}  // namespace serving
}  // namespace cai
