// The format of a cache in 4 bits, and what the kernels that read and write it share.
//
// Pages [n_pages, kv heads, 4, record] of bytes: a record holds 16 tokens of one kv head, so a page's 64 tokens of a
// head are contiguous and any run of whole records is one copy.  In a record, one behind the other: 16 rows of D / 2
// bytes with the keys' codes, 16 rows with the values' codes, and for each token the pairs (s, m) of its key's groups
// of 64 elements, then of its value's: 18 D bytes.  An element is s c + m; s and m are bfloat16 (s in the low half of
// the 32-bit pair), c a code of 4 bits.  Against bfloat16 rows (64 D bytes for 16 tokens) that is 3.56 times less.
//
// m is the group's smallest element rounded down to bfloat16 and s = (largest - m) / 15 rounded up, so that the range
// [m, m + 15 s] holds the group, no code has to be cut off, and an element is off by at most s / 2.  A group whose
// range bfloat16 cannot hold ([m, m + 15 s], not only its elements), or with an element that is not finite, is stored as NaN.
//
// The order of a row's 32-bit words is the order in which the threads of m16n8k16 products take them.  A word has
// eight elements of the head, 8 n .. 8 n + 7 for word n: element 2 i in nibble i and 2 i + 1 in nibble 4 + i, so that
// one shift and one three-input logical operation give a register with two neighbours.
//   keys: rows of A are tokens and the four lanes t of a row share the head's elements: lane t takes the words n with
//     n % 4 = t, which therefore stand side by side (word n at (n % 4) (D / 32) + n / 4): one load of 16 bytes a token.
//   values: rows of A are elements, its columns tokens, and lane group r = lane / 4 takes the words n with n % 8 = r
//     (one of each group of 64): word n at ((n % 8) ^ turn) (D / 64) + n / 8, where turn = 4 for tokens 2, 3 of every
//     four: the four tokens that a half warp reads at once then lie in different banks.
// The token of row i of such a product is kv4_token(i): rows 2 j and 2 j + 1 are tokens of different parity (their keys
// lie in different halves of the banks), and rows 0, 2, 4, 6 (1, 3, 5, 7) are four neighbours in some order.
#pragma once
#include "common.cuh"

#define KV4_PAGE 64        // tokens of a page
#define KV4_TOKENS 16      // tokens of a record
#define KV4_GROUP 64       // elements that share a pair

template <int D>
struct Kv4 {
  static_assert(D == 64 || D == 128, "heads of 64 or 128");
  static constexpr int NG = D / KV4_GROUP;        // groups of a head
  static constexpr int ROW = D / 2;               // bytes of a token's codes
  static constexpr int V_OFF = KV4_TOKENS * ROW;
  static constexpr int PAIR_OFF = 2 * V_OFF;
  static constexpr int PAIR = 8 * NG;             // bytes of a token's pairs: keys' groups, then values'
  static constexpr int RECORD = PAIR_OFF + KV4_TOKENS * PAIR;
  // the place of word n in a key's row, and in the row of the value of a record's token `tok`
  __device__ __forceinline__ static int key_word(int n) { return (n & 3) * (D / 32) + (n >> 2); }
  __device__ __forceinline__ static int value_word(int n, int tok) { return ((n & 7) ^ turn(tok)) * NG + (n >> 3); }
  __device__ __forceinline__ static int turn(int tok) { return (tok & 2) << 1; }
};

// Row i of a product's 16 is this token of the record.
__device__ __forceinline__ int kv4_token(int i) { return (i & 8) + ((i & 1) ? 4 + (((i & 7) >> 1) ^ 1) : ((i & 7) >> 1)); }

// Which page holds a position, or -1: none that the cache has (a position outside the table, or a number that is no
// page's).  Whatever stands in the table, nothing outside the pool is touched.
__device__ __forceinline__ int kv4_page(const int* table, int tile, int max_pages, int n_pages) {
  if ((unsigned)tile >= (unsigned)max_pages) return -1;
  const int p = table[tile];
  return (unsigned)p < (unsigned)n_pages ? p : -1;
}

__device__ __forceinline__ float kv4_s(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float kv4_m(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// Code of element E (0..7) of a word, as a float: the low bits of 2^23's mantissa, less 2^23 (a conversion of whole
// numbers has a quarter of the rate).
template <int E>
__device__ __forceinline__ float kv4_code(uint32_t w) {
  constexpr int AT = ((E & 1) << 4) + ((E >> 1) << 2);
  return __uint_as_float(((w >> AT) & 15u) | 0x4b000000u) - 8388608.f;
}
// The eight elements of a word.
__device__ __forceinline__ void kv4_values(uint32_t w, uint32_t pair, float (&x)[8]) {
  const float s = kv4_s(pair), m = kv4_m(pair);
  x[0] = fmaf(s, kv4_code<0>(w), m), x[1] = fmaf(s, kv4_code<1>(w), m), x[2] = fmaf(s, kv4_code<2>(w), m);
  x[3] = fmaf(s, kv4_code<3>(w), m), x[4] = fmaf(s, kv4_code<4>(w), m), x[5] = fmaf(s, kv4_code<5>(w), m);
  x[6] = fmaf(s, kv4_code<6>(w), m), x[7] = fmaf(s, kv4_code<7>(w), m);
}
