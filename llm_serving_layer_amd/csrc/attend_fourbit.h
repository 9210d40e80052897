// What the kernels of the attention over the 4-bit cache share: tiles, pieces and
// launch arguments.
#pragma once

#include "fourbit.h"

namespace pkv {

constexpr int kTile = 64;          // keys
// A piece: {first token's row in q, tokens, its position, kv_len, first page in
// kv_indices, pages, tile, tiles, partial slot | -1, slot 0, pieces, counter}, then
// the pages of the first four tiles' units.
constexpr int kPieceInts = 28;

constexpr int kTallRows = 128;      // of a tall piece

struct Attend4 {
  const void* q;
  void* out;
  const unsigned char *kpool, *vpool;
  const int32_t *items, *indices;
  int32_t* counters;
  float *part_o, *part_ml;
  int32_t* status;
  int64_t num_blocks, block;
  int32_t n_items, n_kv, groups, head_bytes, pairs, shift, part_rows, count_step;
  uint32_t per_group;                // 2^16 / groups, rounded up: r / groups below 128
  float scale_log2;
};

int run_4bit_tall(const Attend4& a, int32_t head_dim, int32_t dtype, const int32_t* items,
                  int32_t n_items, hipStream_t s);

}  // namespace pkv
