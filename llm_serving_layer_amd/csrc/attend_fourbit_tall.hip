// Attention over the 4-bit cache for many query rows a sequence (prompt chunks): a
// workgroup of four waves takes 128 rows (tokens x heads of a KV head) over all the
// keys they see, 64 at a time. The matrix cores bound it, and beside them the
// softmax's vector work, so a tile's codes become float16 values once for all rows:
//  * each wave takes one unit of 16 keys from memory into registers a tile ahead
//    (a lane its operand's codes, its keys' steps and zeros) and writes zero +
//    step c to LDS: K row by row, V dim by dim, so that both are read as operands
//    16 bytes a lane. Two tiles' buffers, one barrier a tile;
//  * S^T = K Q^T and O^T += V^T P^T by 32x32x16 products, 32 rows a wave; the
//    softmax of a row in its two lanes, its reference moved only when a lane's sum
//    of a tile passes 2^12.
// K and V are rounded to float16 here (2^-12 of a value at most, what a 16-bit cache
// holds of it); with exact codes and the steps applied to the scores and weights, as
// for few rows, 8 x 512 tokens over 1536 (head_dim 64) took 152 us, as here 95
// (640 TFLOP/s).
// Rows of 144 bytes (272 for K at head_dim 128) put the 16 lanes of a 16-byte read on
// different banks.
#include "attend_fourbit.h"

namespace pkv {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// 1024 + c (or 1024 + 16 c) in the halves of w, as numbers less 1024
__device__ __forceinline__ f16x2 code_pair(uint32_t w, uint32_t mask) {
  const f16x2 k{(_Float16)1024.f, (_Float16)1024.f};
  return __builtin_bit_cast(f16x2, (w & mask) | 0x64006400u) - k;
}
__device__ __forceinline__ f16x2 fma2(f16x2 a, f16x2 b, f16x2 c) {
  return __builtin_elementwise_fma(a, b, c);
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void attend_4bit_tall_kernel(Attend4 a) {
  constexpr int NG = D / 64, W = D / 32, NC = D / 16, NB = D / 32;
  constexpr int KS = 2 * D + 16, VS = 2 * kTile + 16;    // bytes of an LDS row
  constexpr int KB = kTile * KS, BUF = KB + D * VS;
  constexpr uint32_t LO = 0x000f000fu, UP = 0x00f000f0u;
  __shared__ __align__(16) unsigned char smem[2 * BUF];
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
  auto halves = [](uint32_t lo, uint32_t hi) {
    return __builtin_bit_cast(f16x2, (lo & 0xffffu) | hi << 16);
  };
  const f16x2 sixteenth{(_Float16)0.0625f, (_Float16)0.0625f};
  // The unit's values into tile buffer `of`. RARE: steps of 4096 on, whose values may
  // round past the largest float16, or NaN: a NaN of V is left out, and its key noted.
  auto stage_as = [&](int of, auto rare) {
    constexpr bool RARE = decltype(rare)::value;
    unsigned char* const buf = smem + of * BUF;
    auto held = [&](f16x2 code, f16x2 step, f16x2 zero) {
      f16x2 v = fma2(code, step, zero);
      if constexpr (RARE) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (__builtin_bit_cast(uint16_t, (_Float16)v[i]) == 0x7c00u) v[i] = (_Float16)kF16Max;
      }
      return __builtin_bit_cast(uint32_t, v);
    };
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t p = kw[w / 2], c = kc[w], c8 = c >> 8;
      const f16x2 step = halves(p >> 16, p >> 16), zero = halves(p, p), s16 = step * sixteenth;
      // elements (0, 4) (1, 5) (2, 6) (3, 7), as Q has them
      const u32x4 v{held(code_pair(c, LO), step, zero), held(code_pair(c, UP), s16, zero),
                    held(code_pair(c8, LO), step, zero), held(code_pair(c8, UP), s16, zero)};
      const int dim = 64 * (w / 2) + 16 * kg + 8 * (w & 1);
      *reinterpret_cast<u32x4*>(buf + (16 * wave + kn) * KS + 2 * dim) = v;
    }
    // V: keys (0, 2), (1, 3) of a quartet; of 16 keys the quartets lie 0 2 1 3, so
    // that a lane's two of a product are neighbours
    const int at = KB + 32 * wave + (kg & 1) * 16 + (kg >> 1) * 8;
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      uint32_t p[4];
      uint32_t none = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[j] = vw[q][j];
        if constexpr (RARE) {
          const bool nan = p[j] >= 0x7c010000u;
          // (bit 4 kg + j of the unit's keys, from the lanes kn = 0)
          const uint64_t b = __builtin_amdgcn_ballot_w64(nan);
          none |= (uint32_t)((b & 1) << j | (b >> 16 & 1) << (4 + j) | (b >> 32 & 1) << (8 + j) |
                             (b >> 48 & 1) << (12 + j));
          p[j] = nan ? 0u : p[j];
        }
      }
      if (lane == 0) nan_keys[of][q][wave] = (uint16_t)none;
      const f16x2 sa = halves(p[0] >> 16, p[2] >> 16), sb = halves(p[1] >> 16, p[3] >> 16);
      const f16x2 za = halves(p[0], p[2]), zb = halves(p[1], p[3]);
      const f16x2 sa16 = sa * sixteenth, sb16 = sb * sixteenth;
#pragma unroll
      for (int b = 2 * q; b < 2 * q + 2; ++b) {
        const uint32_t c = vc[b], c8 = c >> 8;
        const u32x2 lo{held(code_pair(c, LO), sa, za), held(code_pair(c8, LO), sb, zb)};
        const u32x2 up{held(code_pair(c, UP), sa16, za), held(code_pair(c8, UP), sb16, zb)};
        *reinterpret_cast<u32x2*>(buf + at + (32 * b + kn) * VS) = lo;
        *reinterpret_cast<u32x2*>(buf + at + (32 * b + 16 + kn) * VS) = up;
      }
    }
  };
  auto stage = [&](int of) {
    uint32_t top = 0;
#pragma unroll
    for (int q = 0; q < NG; ++q)
      top = max(top, max(max(kw[q], max(vw[q][0], vw[q][1])), max(vw[q][2], vw[q][3])));
    if (__builtin_amdgcn_ballot_w64(top >= 0x6c000000u)) stage_as(of, std::true_type{});
    else stage_as(of, std::false_type{});
  };
  load(0, page(0));

  // Q^T as the B operand: lane (row, g) holds dims 16 c + 8 g .. + 7, scaled by a
  // power of two to a largest element in [128, 256) (a product of 256 elements of
  // +-65504 stays finite), the scale's sign with it.
  const int r = wave * 32 + n;
  const int tok = (int)((uint32_t)r * a.per_group >> 16);
  const bool valid = tok < qn;
  const int qpos = base_pos + (valid ? tok : qn - 1);
  f16x8 qb[NC];
  float f1;
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
        qb[c][i] = (_Float16)(!valid ? 0.f : turn ? -e : e);
      }
  }

  f32x16 o[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b] = f32x16{};
  float ref = -INFINITY, l = 0.f, none[NG] = {};

  stage(0);
  int next = page(1);                // (read a tile ahead of its use)
  if (n_tiles > 1) load(1, next);
  next = page(2);
  __syncthreads();
  for (int t = 0; t < n_tiles; ++t) {
    const unsigned char* buf = smem + (t & 1) * BUF;
    // S^T: s[hf][e] = the row's score with key 64 t + 32 hf + 8 (e / 4) + 4 g + e % 4
    f32x16 s[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) s[hf] = f32x16{};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        s[hf] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
            *reinterpret_cast<const f16x8*>(buf + (32 * hf + n) * KS + 32 * c + 16 * g), qb[c], s[hf],
            0, 0, 0);
    if (kTile * t + kTile - 1 > base_pos) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (kTile * t + 32 * hf + 8 * (e >> 2) + 4 * g + (e & 3) > qpos) s[hf][e] = -INFINITY;
    }
    float ls;
    f16x8 pb[4];
    auto probs = [&](float m) {
      ls = 0.f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[hf][e], f1, -m));
          ls += p;
          // (quartets as V has them: 0 2 1 3)
          pb[2 * hf + (e >> 3)][(e & 4) + ((e & 1) << 1 | (e >> 1 & 1))] = (_Float16)p;
        }
    };
    // (one copy of the weights' code: two took 31 registers more, a third of the waves)
    float m = ref;
    for (int again = 0;; ++again) {
      probs(m);
      if (again || !__builtin_amdgcn_ballot_w64(!(ls <= 4096.f))) break;
      float mx = -INFINITY;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[hf][e]);
      m = fmaxf(ref, max_x32(mx) * f1);
      const float alpha = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref - m);
      ref = m;
      m = m == -INFINITY ? 0.f : m;
      l *= alpha;
#pragma unroll
      for (int b = 0; b < NB; ++b) o[b] *= alpha;
    }
    l += ls;
    // the next tile into the other buffer, the one after it on its way
    if (t + 1 < n_tiles) {
      stage((t + 1) & 1);
      if (t + 2 < n_tiles) load(t + 2, next);
      next = page(t + 3);
    }
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int b = 0; b < NB; ++b)
        o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
            *reinterpret_cast<const f16x8*>(buf + KB + (32 * b + n) * VS + 32 * kb + 16 * g), pb[kb],
            o[b], 0, 0, 0);
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
  if (!valid) return;
  const float inv = 1.f / l;
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
  if (grid > 0x7fffffffLL) return fail(PKV_ERR_INVALID, "too many row tiles");
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
