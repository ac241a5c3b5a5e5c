// Layout of the 8-bit key/value cache of one layer, shared by the kernels that write, read and attend it.
//
//   scales  float32 [n_seq][n_heads][blocks][2]   (keys, values), each an exact power of two; then, 256-byte aligned,
//   tiles   [n_seq][n_heads][blocks] x 16 KiB     8 KiB of key codes, 8 KiB of value codes
//
// A block is 64 consecutive tokens; the last one of a sequence is filled up with zero codes.  Inside a tile the codes
// stand in the order in which the attention kernel's lanes hold them as matrix operands, so that a wave fetches a tile
// with sixteen fully contiguous 1-KiB loads straight into registers (no LDS, no transposition, no barrier):
//   keys    piece (kb, j), kb 0..1, j 0..3: lane l holds 16 bytes = key 32 kb + (l & 31), dims 64 (l >> 5) + 16 j + 0..15
//   values  piece (db, kb), db 0..3, kb 0..1: lane l holds 16 bytes = dim 32 db + (l & 31), word w (0..3) = keys
//           32 kb + 8 w + 4 (l >> 5) + 0..3   (the order in which the score registers of a lane hold those keys)
#pragma once
#include "common.h"

constexpr int KV8_TOKENS = 64;
constexpr int KV8_HD = 128;
constexpr int KV8_CODES = KV8_TOKENS * KV8_HD;     // codes of one operand of a tile
constexpr int KV8_TILE = 2 * KV8_CODES;

inline int64_t kv8_blocks(int64_t seq_len) { return (seq_len + KV8_TOKENS - 1) / KV8_TOKENS; }
inline size_t kv8_scale_bytes(int64_t n_tiles) { return ((size_t)n_tiles * 8 + 255) & ~(size_t)255; }

// byte offset of the code of (key, dim) inside the keys' / the values' half of a tile
__device__ __forceinline__ int kv8_key_offset(int key, int dim) {
    return (((key >> 5) * 4 + ((dim >> 4) & 3)) * 64 + (dim >> 6) * 32 + (key & 31)) * 16 + (dim & 15);
}
__device__ __forceinline__ int kv8_value_offset(int key, int dim) {
    return (((dim >> 5) * 2 + (key >> 5)) * 64 + ((key >> 2) & 1) * 32 + (dim & 31)) * 16 + ((key >> 3) & 3) * 4 + (key & 3);
}
