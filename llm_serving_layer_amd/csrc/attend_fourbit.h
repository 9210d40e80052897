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

// Words from here on are a NaN group's.
constexpr uint32_t kNoStep = 0x7c000000u;

// The largest of the lanes up to this one's.
__device__ __forceinline__ uint32_t scan_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));  // row_shr
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  // row_bcast:15 into rows 1 and 3, row_bcast:31 into 2 and 3
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return v;
}

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
