// The paged cache of keys and values in 4 or 8 bits: what a group of values is held as, and where it lies.
//
// A group x (32 neighbouring elements of a key, the whole head of a value) is held as codes c, a step s and an offset z,
// both bfloat16, and stands for z + s (c - H), H = 2^(bits - 1):
//     z = bf16((H max x + (H - 1) min x) / (2H - 1))
//     s = max((max x - z) / (H - 1), (z - min x) / H), rounded to float32 and then up to bfloat16
//     c = round((x - z) / s) + H, ties to even, within 0 .. 2H - 1
// The step is chosen after the offset has been rounded, and rounded up, so every x lies within half a step of a value that
// is held, whatever the rounding of z.  A group with an infinity or a NaN in it has a NaN for its step and its offset.
//
// One page: bytes [key/value heads][head bytes]; one head of a page of P tokens (P a multiple of 8, D of 32):
//     keys    [P][4][D / 32][8]  codes: element 32 g + 8 j + e at [j][g][e], so that the lanes 16 j .. 16 j + 15 of a matrix
//             instruction read their elements of all the groups in one piece.  With 4 bits, eight codes are a word in which
//             element e has the four bits from 4 (e / 2 + 4 (e % 2)) on: a shift and a mask leave two neighbours in the halves.
//     values  [P / 8][D][8]      codes, eight tokens of a dimension together (one operand of the matrix instruction); with 4
//             bits [P / 8][D / 2][8] bytes, an even dimension in the low half of a byte, the next one in the high half, token
//             t of eight in byte (0, 2, 1, 3, 4, 6, 5, 7)[t]: every byte belongs to one token, so tokens are written without
//             reading what is there, and again a shift and a mask leave two neighbours.
//     words   [P][D / 32] of the keys, then [P] of the values: s in a word's upper half, z in its lower
#pragma once
#include "common.h"

__host__ __device__ constexpr long quant_token_bytes(int head_dim, int bits) { return 2l * (head_dim * bits / 8) + head_dim / 32 * 4 + 4; }

// Where the parts of one head of a page begin, in bytes from the head's first.
struct QuantHead {
  long values, key_words, value_words, bytes;
};
__host__ __device__ __forceinline__ QuantHead quant_head(int page_size, int head_dim, int bits) {
  QuantHead h;
  h.values = (long)page_size * (head_dim * bits / 8);
  h.key_words = 2 * h.values;
  h.value_words = h.key_words + (long)page_size * (head_dim / 32) * 4;
  h.bytes = h.value_words + (long)page_size * 4;
  return h;
}

__device__ __forceinline__ int quant_place(int token) {  // byte of token t of eight among those of a pair of dimensions (4 bits)
  return (token & 4) | ((token & 1) << 1) | ((token >> 1) & 1);
}

__device__ __forceinline__ float word_step(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float word_offset(uint32_t w) { return __uint_as_float(w << 16); }

// The largest head size that the kernels take.
#define QUANT_MAX_DIM 256

// What every entry point asks of the sizes.
#define QUANT_REQUIRE_SIZES(what)                                                                                              \
  CWM_REQUIRE(bits == 4 || bits == 8, what ": a cache holds 4 or 8 bits a value, not %d", bits);                               \
  CWM_REQUIRE(head_dim % 32 == 0 && head_dim >= 32 && head_dim <= QUANT_MAX_DIM, what ": head_dim %d is no multiple of 32 up to %d", \
              head_dim, QUANT_MAX_DIM);                                                                                        \
  CWM_REQUIRE(page_size > 0 && page_size % 8 == 0, what ": page size %d must be a multiple of 8", page_size);                  \
  CWM_REQUIRE(num_pages > 0 && table_width > 0 && n_kv_heads > 0, what ": bad cache geometry")
