// Attention over the 4-bit cache for many query rows a sequence (prompt chunks): a
// workgroup of four waves takes 128 rows (tokens x heads of a KV head) over all the
// keys they see, 64 at a time. The softmax's vector work bounds it, and beside it the
// matrix cores, so a tile's codes become operands once for all rows:
//  * each wave takes one unit of 16 keys from memory into registers a tile ahead
//    (a lane its operand's codes, its keys' words) and writes to LDS: K's codes as
//    float16 numbers c 2^-24, row by row, V's as (c - 7.5) 2^-9, dim by dim, so that
//    both are read as operands 16 bytes a lane; and the words. Two tiles' buffers, one
//    barrier a tile;
//  * S^T = K Q^T and O^T += V^T P^T by 32x32x16 products, 32 rows a wave; a score is
//    sum_g step_g (q . c)_g + zero_g sum q, exact but for 32-bit sums; the softmax of a
//    row in its two lanes, its reference moved only when a score passes it by 2^12;
//  * P is p step, rounded to float16 once (2^-11 of it), against c - 7.5, and in 32
//    bits p zero + 7.5 p step. With 2^E at least the largest step that the row has seen,
//    p counts 2^-E more, so that p step stays within float16.
// 8 x 512 tokens over 1536, head_dim 64, 8 KV heads of 4: 122 us, 490 TFLOP/s (as wide
// pieces 150). With keys and values rounded to float16 in LDS and p beside them it took
// 95, but three roundings of 2^-11 added 1.4 times the output's own error; this one adds
// as much as it.
// Rows of 144 bytes (272 for K at head_dim 128) put the 16 lanes of a 16-byte read on
// different banks.
#include "attend_fourbit.h"

namespace pkv {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float step_of(uint32_t w) { return (float)f16_bits(w >> 16); }
__device__ __forceinline__ float zero_of(uint32_t w) { return (float)f16_bits(w & 0xffffu); }

template <typename T, int D>
__global__ __launch_bounds__(256, (D == 64 ? 3 : 2)) void attend_4bit_tall_kernel(Attend4 a) {
  constexpr int NG = D / 64, W = D / 32, NC = D / 16, NB = D / 32;
  // keys of a step, in 32: all of a tile's, or half where the registers hold no more
  // (head_dim 64 in halves: 131 us for 122; 128 in whole tiles: 298 for 267)
  constexpr int NH = D == 64 ? 2 : 1;
  constexpr int KS = 2 * D + 16, VS = 2 * kTile + 16;    // bytes of an LDS row
  constexpr int KB = kTile * KS, BUF = KB + D * VS;
  constexpr uint32_t LO = 0x000f000fu, UP = 0x00f000f0u;
  __shared__ __align__(16) unsigned char smem[2 * BUF];
  __shared__ __align__(16) uint32_t words[2][2][NG][kTile];   // a tile's, of K and of V
  __shared__ __align__(16) uint32_t tops[2][4];          // its units' largest words of V
  __shared__ float row_top[256];     // a lane's row's E, from the first tile seen in part
  __shared__ __align__(8) uint16_t nan_keys[2][NG][4];   // a tile's keys whose V is NaN

  // (as in the pieces' kernel: a tile's heads on one XCD)
  const int x = blockIdx.x & 7, y = blockIdx.x >> 3;
  const int item = (y / a.n_kv) * 8 + x, h = y % a.n_kv;
  if (item >= a.n_items) return;
  const int32_t* it = a.items + (int64_t)item * kPieceInts;
  const int q0 = it[0], qn = it[1], base_pos = it[2], kv_len = it[3], pbase = it[4],
            n_pages = it[5], n_tiles = it[7];
  const int G = a.groups, Hq = a.n_kv * G;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = lane >> 4, kn = lane & 15;    // of a unit's layout
  const int g = lane >> 5, n = lane & 31;      // of a product's

  // the wave's unit of a tile, on its way
  typedef uint32_t Words __attribute__((ext_vector_type(W)));
  const int shift = a.shift, mask = (1 << shift) - 1, ps = 16 << shift;
  const uint32_t k_off = h * a.head_bytes + kn * (D / 2) + kg * (D / 8);
  const uint32_t v_off = h * a.head_bytes + lane * (D / 8);
  Words kc, vc;
  uint32_t kw[NG];
  u32x4 vw[NG];
  uint32_t worst = 0;
  auto page = [&](int t) {
    return __builtin_amdgcn_readfirstlane(
        a.indices[pbase + min((4 * t + wave) >> shift, n_pages - 1)]);
  };
  auto load = [&](int t, int id) {
    const bool bad = (uint64_t)(int64_t)id >= (uint64_t)a.num_blocks;
    worst |= bad;
    const int sub = (4 * t + wave) & mask;
    const uint64_t block = (uint64_t)(uint32_t)(bad ? 0 : id) * (uint32_t)a.block;
    const unsigned char* kb = a.kpool + block;
    const unsigned char* vb = a.vpool + block;
    kc = *reinterpret_cast<const Words*>(kb + sub * 8 * D + k_off);
    vc = *reinterpret_cast<const Words*>(vb + sub * 8 * D + v_off);
    const int key = kTile * t + 16 * wave;      // the unit's first
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const uint32_t at = a.pairs + ((h * NG + q) * ps + sub * 16) * 4;
      kw[q] = *reinterpret_cast<const uint32_t*>(kb + at + kn * 4);
      vw[q] = *reinterpret_cast<const u32x4*>(vb + at + kg * 16);
    }
    // keys past the end and of pages out of range: zeros
    if (bad || key + 16 > kv_len) {
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        if (bad || key + kn >= kv_len) kw[q] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (bad || key + 4 * kg + j >= kv_len) vw[q][j] = 0;
      }
    }
  };
  // The unit into tile buffer `of`. A word of V that is NaN is left out, its key noted.
  auto stage = [&](int of) {
    unsigned char* const buf = smem + of * BUF;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      // elements (0, 4) (1, 5) (2, 6) (3, 7), as Q has them; the second and fourth
      // pair 16 times as large
      const uint32_t c = kc[w], c8 = c >> 8;
      const int dim = 64 * (w / 2) + 16 * kg + 8 * (w & 1);
      *reinterpret_cast<u32x4*>(buf + (16 * wave + kn) * KS + 2 * dim) =
          u32x4{c & LO, c & UP, c8 & LO, c8 & UP};
    }
    uint32_t top = 0;
#pragma unroll
    for (int q = 0; q < NG; ++q)
      top = max(top, max(max(vw[q][0], vw[q][1]), max(vw[q][2], vw[q][3])));
    uint32_t none[NG] = {};
    if (__builtin_amdgcn_ballot_w64(top >= kNoStep)) {
      top = 0;
#pragma unroll
      for (int q = 0; q < NG; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool nan = vw[q][j] >= kNoStep;
          // (bit 4 kg + j of the unit's keys, from the lanes kn = 0)
          const uint64_t b = __builtin_amdgcn_ballot_w64(nan);
          none[q] |= (uint32_t)((b & 1) << j | (b >> 16 & 1) << (4 + j) | (b >> 32 & 1) << (8 + j) |
                                (b >> 48 & 1) << (12 + j));
          vw[q][j] = nan ? 0u : vw[q][j];
          top = max(top, vw[q][j]);
        }
    }
    const uint32_t unit_top = max(max(__builtin_amdgcn_readlane(top, 0), __builtin_amdgcn_readlane(top, 16)),
                                  max(__builtin_amdgcn_readlane(top, 32), __builtin_amdgcn_readlane(top, 48)));
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      if (lane < 16) words[of][0][q][16 * wave + kn] = kw[q];
      if (kn == 0) *reinterpret_cast<u32x4*>(&words[of][1][q][16 * wave + 4 * kg]) = vw[q];
      if (lane == 0) nan_keys[of][q][wave] = (uint16_t)none[q];
    }
    if (lane == 0) tops[of][wave] = unit_top;
    // V: keys (0, 2), (1, 3) of a quartet; of 16 keys the quartets lie 0 2 1 3, so
    // that a lane's two of a product are neighbours
    const int at = KB + 32 * wave + (kg & 1) * 16 + (kg >> 1) * 8;
    auto middle = [](uint32_t codes, float unit) {    // (c - 7.5) 2^-9 of c unit 2^-24
      const _Float16 f = (_Float16)(0x1p15f / unit), m = (_Float16)(-7.5f * 0x1p-9f);
      return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(
          __builtin_bit_cast(f16x2, codes), f16x2{f, f}, f16x2{m, m}));
    };
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t c = vc[b], c8 = c >> 8;
      *reinterpret_cast<u32x2*>(buf + at + (32 * b + kn) * VS) =
          u32x2{middle(c & LO, 1.f), middle(c8 & LO, 1.f)};
      *reinterpret_cast<u32x2*>(buf + at + (32 * b + 16 + kn) * VS) =
          u32x2{middle(c & UP, 16.f), middle(c8 & UP, 16.f)};
    }
  };
  load(0, page(0));

  // Q^T as the B operand: lane (row, g) holds dims 16 c + 8 g .. + 7, scaled by a
  // power of two to a largest element in [128, 256) (a product of 256 elements of
  // +-65504 stays finite), the scale's sign with it; the elements whose codes count 16
  // times as much a 16th. qs: a group's sum, in a product's unit of 2^-24.
  const int r = wave * 32 + n;
  const int tok = (int)((uint32_t)r * a.per_group >> 16);
  const bool valid = tok < qn;
  const int qpos = base_pos + (valid ? tok : qn - 1);
  f16x8 qb[NC];
  float f1, qs[NG] = {};
  {
    typedef T TV __attribute__((ext_vector_type(8)));
    const T* row = reinterpret_cast<const T*>(a.q) +
                   ((int64_t)(q0 + (valid ? tok : 0)) * Hq + h * G + (valid ? r - tok * G : 0)) * D;
    TV v[NC];
    float mx = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      v[c] = *reinterpret_cast<const TV*>(row + 16 * c + 8 * g);
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, __builtin_fabsf(Elem<T>::to_f(v[c][i])));
    }
    mx = max_x32(mx);
    const int k = mx > 0.f && mx < INFINITY ? 8 - __builtin_amdgcn_frexp_expf(mx) : 0;
    f1 = __builtin_amdgcn_ldexpf(__builtin_fabsf(a.scale_log2), -k);
    f1 = f1 < 0x1p-120f ? 0x1p-120f : f1;
    const bool turn = a.scale_log2 < 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = __builtin_amdgcn_ldexpf(Elem<T>::to_f(v[c][(i >> 1) + 4 * (i & 1)]), k);
        const _Float16 x = (_Float16)(!valid ? 0.f : turn ? -e : e);
        qs[c / 4] += (float)x;
        qb[c][i] = (i & 2) ? x * (_Float16)0.0625f : x;
      }
    f1 *= 0x1p24f;
#pragma unroll
    for (int q = 0; q < NG; ++q) qs[q] = sum_x32(qs[q]) * 0x1p-24f;
  }

  f32x16 o[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b] = f32x16{};
  float ref = -INFINITY, l = 0.f, none[NG] = {};
  float zeros[NG] = {}, steps[NG] = {};   // sums of p zero, p step
  int whole_top = -30;               // E, all rows' until a tile is seen in part

  stage(0);
  int next = page(1);                // (read a tile ahead of its use)
  if (n_tiles > 1) load(1, next);
  next = page(2);
  __syncthreads();
  for (int t = 0; t < n_tiles; ++t) {
    const unsigned char* buf = smem + (t & 1) * BUF;
    const auto& wk = words[t & 1][0];
    const auto& wv = words[t & 1][1];
    // a larger step than any that the rows have seen: the sums in its unit
    const bool in_part = kTile * t + kTile - 1 > base_pos;     // (by some row)
    const u32x4 tile_tops = *reinterpret_cast<const u32x4*>(tops[t & 1]);
    const uint32_t word = __builtin_amdgcn_readfirstlane(
        max(max(tile_tops[0], tile_tops[1]), max(tile_tops[2], tile_tops[3])));
    const int now =
        word >= 0x10000u && !in_part ? __builtin_amdgcn_frexp_expf(step_of(word)) : whole_top;
    float by = 1.f;                  // what the sums so far count now
    bool less = now > whole_top;
    if (less) {
      by = __builtin_amdgcn_ldexpf(1.f, whole_top - now);
      ref += (float)(now - whole_top);
      whole_top = now;
    }
#pragma unroll
    for (int h0 = 0; h0 < 2; h0 += NH) {
      // s[hf][e] = the row's score with key 64 t + 32 (h0 + hf) + 8 (e / 4) + 4 g + e % 4
      f32x16 s[NH];
#pragma unroll
      for (int hf = 0; hf < NH; ++hf) {
        f32x16 acc[NG];
#pragma unroll
        for (int q = 0; q < NG; ++q) acc[q] = f32x16{};
#pragma unroll
        for (int c = 0; c < NC; ++c)
          acc[c / 4] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              *reinterpret_cast<const f16x8*>(buf + (32 * (h0 + hf) + n) * KS + 32 * c + 16 * g),
              qb[c], acc[c / 4], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int q = 0; q < NG; ++q) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(&wk[q][32 * (h0 + hf) + 8 * j + 4 * g]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int e = 4 * j + i;
              const float z = __builtin_fmaf(zero_of(w[i]), qs[q], q ? s[hf][e] : 0.f);
              s[hf][e] = __builtin_fmaf(step_of(w[i]), acc[q][e], z);
            }
          }
      }
      float top = (float)whole_top;
      if (in_part) {
        const int key = kTile * t + 32 * h0;
#pragma unroll
        for (int hf = 0; hf < NH; ++hf)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (key + 32 * hf + 8 * (e >> 2) + 4 * g + (e & 3) > qpos) s[hf][e] = -INFINITY;
        // (the row's E, from its own keys in such tiles)
        if (h0 || (t > 0 && kTile * t - 1 > base_pos)) top = row_top[threadIdx.x];
        if (h0 == 0) {
          uint32_t seen = 0;
#pragma unroll
          for (int q = 0; q < NG; ++q) seen = max(seen, wv[q][lane]);
          const int last = qpos - kTile * t;
          seen = (uint32_t)__shfl((int)scan_max(seen), min(max(last, 0), kTile - 1), 64);
          const float more =
              last < 0 || seen < 0x10000u
                  ? 0.f
                  : fmaxf((float)__builtin_amdgcn_frexp_expf(step_of(seen)) - top, 0.f);
          by = __builtin_amdgcn_exp2f(-more);
          ref += more;
          top += more;
          row_top[threadIdx.x] = top;
          less = true;
        }
      }
      // (looking at the largest score first keeps the scores' registers for the weights)
      float mx = -INFINITY;
#pragma unroll
      for (int hf = 0; hf < NH; ++hf)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[hf][e]);
      mx = __builtin_fmaf(mx, f1, top);
      if (__builtin_amdgcn_ballot_w64(!(mx - ref <= 12.f))) {
        const float m = fmaxf(ref, max_x32(mx));
        by *= m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref - m);
        less = true;
        ref = m;
      }
      if (less) {
        l *= by;
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          zeros[q] *= by;
          steps[q] *= by;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] *= by;
        less = false;
        by = 1.f;
      }
      f16x8 pb[NG][2 * NH];
      const float m = ref == -INFINITY ? 0.f : ref;
#pragma unroll
      for (int hf = 0; hf < NH; ++hf)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[hf][4 * j + i], f1, -m));
            l += p[i];
          }
#pragma unroll
          for (int q = 0; q < NG; ++q) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(&wv[q][32 * (h0 + hf) + 8 * j + 4 * g]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              zeros[q] = __builtin_fmaf(p[i], zero_of(w[i]), zeros[q]);
              steps[q] = __builtin_fmaf(p[i], step_of(w[i]), steps[q]);
              // (quartets as V has them: 0 2 1 3)
              pb[q][2 * hf + (j >> 1)][(4 * j & 4) + ((i & 1) << 1 | (i >> 1 & 1))] =
                  (_Float16)__builtin_fmaf(p[i], step_of(w[i]), 0.f);
            }
          }
        }
      // the next tile into the other buffer, the one after it on its way
      if (h0 == 0 && t + 1 < n_tiles) {
        stage((t + 1) & 1);
        if (t + 2 < n_tiles) load(t + 2, next);
        next = page(t + 3);
      }
#pragma unroll
      for (int kb = 0; kb < 2 * NH; ++kb)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              *reinterpret_cast<const f16x8*>(buf + KB + (32 * b + n) * VS + 64 * h0 + 32 * kb + 16 * g),
              pb[b / 2][kb], o[b], 0, 0, 0);
    }
    // a row that sees a key whose V is NaN gets NaN, at the end
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const uint64_t keys = *reinterpret_cast<const uint64_t*>(nan_keys[t & 1][q]);
      if (__builtin_amdgcn_readfirstlane((uint32_t)keys | (uint32_t)(keys >> 32))) {
        const int seen = qpos - kTile * t;     // the last one
        const uint64_t mine = seen < 0 ? 0 : seen >= 63 ? keys : keys & ((2ull << seen) - 1);
        none[q] = mine ? NAN : none[q];
      }
    }
    __syncthreads();
  }
  if (worst && lane == 0) flag(a.status, PKV_STATUS_BAD_PAGE);
  l = sum_x32(l);
#pragma unroll
  for (int q = 0; q < NG; ++q) none[q] += sum_x32(__builtin_fmaf(7.5f, steps[q], zeros[q])) / l;
  if (!valid) return;
  const float inv = 512.f / l;
  typedef T TV4 __attribute__((ext_vector_type(4)));
  T* row = reinterpret_cast<T*>(a.out) + ((int64_t)(q0 + tok) * Hq + h * G + r - tok * G) * D + 4 * g;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      TV4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)__builtin_fmaf(o[b][4 * j + e], inv, none[b / 2]);
      *reinterpret_cast<TV4*>(row + 32 * b + 8 * j) = v;
    }
}

int run_4bit_tall(const Attend4& args, int32_t head_dim, int32_t dtype, const int32_t* items,
                  int32_t n_items, hipStream_t s) {
  Attend4 a = args;
  a.items = items;
  a.n_items = n_items;
  const int64_t grid = (int64_t)((n_items + 7) / 8) * a.n_kv * 8;
  if (!launchable(grid, 256)) return fail(PKV_ERR_INVALID, "too many row tiles");
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, s, a);
  };
  if (dtype == PKV_DTYPE_F16) {
    if (head_dim == 64) go(attend_4bit_tall_kernel<_Float16, 64>);
    else go(attend_4bit_tall_kernel<_Float16, 128>);
  } else {
    if (head_dim == 64) go(attend_4bit_tall_kernel<__bf16, 64>);
    else go(attend_4bit_tall_kernel<__bf16, 128>);
  }
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

}  // namespace pkv
