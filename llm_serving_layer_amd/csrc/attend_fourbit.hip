// Attention over the 4-bit cache (format: fourbit.h) on gfx950 matrix cores, for
// head_dim 64 and 128 and fp16 or bf16 queries.
//
// With k = zero + step c in each group q of 64 dims,
//   q . k = sum_q step_q (q_q . c_q) + zero_q sum(q_q),
// and with the softmax weights p, sum_t p_t v_t = sum_t (p_t step_t) c_t +
// sum_t p_t zero_t: the matrix cores multiply by the codes as they are. A code in
// the low bits of a 16-bit half is a subnormal float16 (c 2^-24, or c 2^-20 where
// it lies four bits up), which they take exactly; so a word of eight codes becomes
// an operand by four ANDs and a shift, and the powers of two go into the query's
// elements, the softmax's factor and the output. Steps and zeros enter in 32 bits
// once per key and group, not per element.
//
// A workgroup of four waves takes one KV head of a piece: up to 16 RT query rows
// (tokens x heads of a sequence) over a run of tiles of 64 keys, which the waves
// take in turn, each with a softmax of its own; they meet in LDS at the end. A
// tile is four units of 16 keys (page rows); lane 16 g + n:
//  * S^T = K Q^T (16x16x32): K codes as the A operand straight from memory (lane:
//    key n, dims 16 g .. of each group), so lane (g, n) gets scores of query row n
//    and keys 4 g .. 4 g + 3 of a unit;
//  * O^T += V^T P^T: V codes as the A operand (lane: dim n, keys 4 g ..), the
//    lane's own probabilities as the B operand. All of a row's state lies in its
//    lanes.
// Few rows leave most of the 16 columns of S^T idle, so they become classes: with
// at most 4 (8) rows, columns n / 4 (n / 8) are 4 (2) classes, and class c takes
// the units u = c (mod classes) alone: Q is zero elsewhere, and one accumulator
// gathers four units' scores. A lane then does the softmax of 4 keys a tile, not
// 16, and the classes meet at the end like the waves.
//
// Each wave loads the next tile's codes (16 bytes a lane at head_dim 128) while it
// computes one, page ids two tiles ahead; the words with steps and zeros, a lane a
// key, go through the wave's LDS. Long sequences are cut into pieces of several
// workgroups, whose partial results the last of them to arrive merges.
//
// The running reference of the softmax moves lazily: only when a lane's sum of a
// tile's probabilities passes 2^12, or when a step of V outgrows the power of two
// 2^e that keeps p step within float16 (p 2^e against the reference).
#include <algorithm>
#include <exception>
#include <vector>

#include "fourbit.h"

namespace pkv {

int check_seq_pages(int32_t i, int32_t np, int32_t kv, int32_t last, int32_t ps);
int check_4bit(int32_t n_kv, int32_t d, int32_t ps);
int run_4bit_any(const pkv_4bit& b, const void* q, void* out, const void* k_pool,
                 const void* v_pool, float scale, hipStream_t s);

constexpr int kTile = 64;          // keys
constexpr int kPieceInts = 8;      // {seq, first token, tokens, tile, tiles, slot | -1, slot 0, pieces}
constexpr int kWaves = 4;

struct Attend4 {
  const void* q;
  void* out;
  const unsigned char *kpool, *vpool;
  const int32_t *items, *cu_q, *indptr, *indices, *kv_lens;
  int32_t* counters;
  float *part_o, *part_ml;
  int32_t* status;
  int64_t num_blocks, block;
  int32_t n_items, n_kv, groups, head_bytes, pairs, shift, part_rows;
  float scale_log2;
};

// Per wave: the steps and zeros of a tile's K and V ([K | V][group][key]).
template <int D> constexpr int kPairInts = 2 * (D / 64) * kTile;

template <typename T, int D, int RT, int NCL>
__global__ __launch_bounds__(64 * kWaves) void attend_4bit_kernel(Attend4 a) {
  constexpr int NG = D / 64;         // groups
  constexpr int W = D / 32;          // words of codes a lane takes of a unit
  constexpr int NT = D / 16;         // output tiles of 16 dims
  constexpr int RC = 16 / NCL;       // rows of a class
  constexpr int UPL = 4 / NCL;       // units of a tile whose scores a lane holds
  constexpr int ROWS = RT * 16;      // columns of S^T
  constexpr int OROWS = NCL > 1 ? RC : ROWS;
  constexpr int OP = D + 4;          // floats of a row of the merge's LDS
  static_assert(RT == 1 || NCL == 1, "classes are for few rows");
  __shared__ __align__(16) uint32_t pair_lds[kWaves * kPairInts<D>];
  __shared__ __align__(16) float o_lds[kWaves * ROWS * OP];
  __shared__ float m_lds[kWaves * ROWS], l_lds[kWaves * ROWS];
  __shared__ int arrived;

  // Eight XCDs take workgroups in turn; a piece's heads go to one of them, where
  // they share the lines that hold steps and zeros of two heads.
  const int x = blockIdx.x & 7, y = blockIdx.x >> 3;
  const int item = (y / a.n_kv) * 8 + x, h = y % a.n_kv;
  if (item >= a.n_items) return;
  const int32_t* it = a.items + (int64_t)item * kPieceInts;
  const int seq = it[0], qs = it[1], qn = it[2], tile0 = it[3], n_tiles = it[4], slot = it[5];
  const int q0 = a.cu_q[seq], q_len = a.cu_q[seq + 1] - q0;
  const int kv_len = a.kv_lens[seq], pbase = a.indptr[seq];
  const int n_pages = a.indptr[seq + 1] - pbase;
  const int base_pos = kv_len - q_len + qs;      // the piece's first token's position
  const int G = a.groups, Hq = a.n_kv * G;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, g = lane >> 4, n = lane & 15;
  const int cls = NCL > 1 ? n / RC : 0;

  // Queries: scaled by a power of two that brings the row's largest element to
  // [1024, 2048), exactly (bf16 too, but for elements 2^-35 of the largest), and
  // turned over for a negative scale; in the order of an operand's codes, where
  // every other one is 16 times its value.
  f16x8 qop[RT][NCL][2 * NG];
  float qsum[RT][NG], f1[RT];
  int qpos[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = NCL > 1 ? n % RC : rt * 16 + n;
    const int tok = r / G;
    const bool valid = tok < qn;
    qpos[rt] = base_pos + (valid ? tok : qn - 1);
    typedef T TV __attribute__((ext_vector_type(8)));
    const T* row = reinterpret_cast<const T*>(a.q) +
                   ((int64_t)(q0 + qs + (valid ? tok : 0)) * Hq + h * G + r % G) * D + 16 * g;
    float v[2 * NG][8], mx = 0.f;
#pragma unroll
    for (int w = 0; w < 2 * NG; ++w) {
      const TV t = *reinterpret_cast<const TV*>(row + (w >> 1) * 64 + (w & 1) * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[w][i] = valid ? Elem<T>::to_f(t[i]) : 0.f;
        mx = fmaxf(mx, __builtin_fabsf(v[w][i]));
      }
    }
    mx = max_x32(max_x16(mx));
    const bool scaled = mx > 0.f && mx < INFINITY;
    const int k = scaled ? 11 - __builtin_amdgcn_frexp_expf(mx) : 0;
    const float sign = a.scale_log2 < 0.f ? -1.f : 1.f;
    // (a scale of 0: small enough to change nothing, and no 0 x inf at masks)
    f1[rt] = __builtin_amdgcn_ldexpf(__builtin_fabsf(a.scale_log2), 24 - k);
    f1[rt] = f1[rt] < 0x1p-120f ? 0x1p-120f : f1[rt];
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      float sum = 0.f;
#pragma unroll
      for (int w = 2 * q; w < 2 * q + 2; ++w) {
        f16x8 op;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = (i >> 1) + 4 * (i & 1);       // elements 0 4 1 5 2 6 3 7
          const bool up = (i >> 1) & 1;               // codes four bits up
          op[i] = (_Float16)(__builtin_amdgcn_ldexpf(v[w][e], k) * sign * (up ? 0.0625f : 1.f));
          sum += (float)op[i] * (up ? 16.f : 1.f);
        }
#pragma unroll
        for (int c = 0; c < NCL; ++c) qop[rt][c][w] = NCL == 1 || c == cls ? op : f16x8{};
      }
      qsum[rt][q] = sum_x32(sum_x16(sum)) * 0x1p-24f;
    }
  }

  // a tile on its way
  struct Tile {
    uint32_t k[4][W], v[4][W];
    uint32_t kp[NG], vp[NG];
    int id;
  };
  const int shift = a.shift, mask = (1 << shift) - 1;    // units of a page
  auto load_id = [&](int t) {      // the page of lane group g's unit of tile t
    return a.indices[pbase + min((4 * t + g) >> shift, n_pages - 1)];
  };
  const int unit_bytes = 8 * D;
  const int k_off = h * a.head_bytes + n * (D / 2) + g * (D / 8);
  const int v_off = h * a.head_bytes + lane * (D / 8);
  const int ps = 16 << shift;
  typedef uint32_t Words __attribute__((ext_vector_type(W)));
  auto load = [&](Tile& x, int t, int id) {
    x.id = id;
    const int ok = (uint64_t)(int64_t)id < (uint64_t)a.num_blocks ? id : 0;
    const int64_t mine = (int64_t)ok * a.block + a.pairs +
                         ((h * NG) * ps + ((4 * t + g) & mask) * 16 + n) * 4;
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      x.kp[q] = __builtin_nontemporal_load(
          reinterpret_cast<const uint32_t*>(a.kpool + mine + q * ps * 4));
      x.vp[q] = __builtin_nontemporal_load(
          reinterpret_cast<const uint32_t*>(a.vpool + mine + q * ps * 4));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t at = (int64_t)__builtin_amdgcn_readlane(ok, 16 * u) * a.block +
                         ((4 * t + u) & mask) * unit_bytes;
      const Words kw = __builtin_nontemporal_load(
          reinterpret_cast<const Words*>(a.kpool + at + k_off));
      const Words vw = __builtin_nontemporal_load(
          reinterpret_cast<const Words*>(a.vpool + at + v_off));
#pragma unroll
      for (int w = 0; w < W; ++w) {
        x.k[u][w] = kw[w];
        x.v[u][w] = vw[w];
      }
    }
  };

  f32x4 o[RT][NT];
  float ref[RT], l[RT], zo[RT][NG];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int i = 0; i < NT; ++i) o[rt][i] = f32x4{};
#pragma unroll
    for (int q = 0; q < NG; ++q) zo[rt][q] = 0.f;
    ref[rt] = -INFINITY;
    l[rt] = 0.f;
  }
  uint32_t cap = 0;                  // the largest step (a word's) that 2^e allows
  int e = 0;
  float limit = 4096.f;              // 2^12 2^e
  uint32_t worst = 0;                // any page id out of range
  uint32_t* const pw = pair_lds + wave * kPairInts<D>;
  const uint32_t LO = 0x000f000fu, UP = 0x00f000f0u;

  auto compute = [&](Tile& x, int t) {
    // steps and zeros; none for keys past the end and for pages out of range,
    // which read as zeros
    const bool bad = (uint64_t)(int64_t)x.id >= (uint64_t)a.num_blocks;
    const bool live = kTile * t + lane < kv_len && !bad;
    worst |= bad;
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      x.kp[q] = live ? x.kp[q] : 0u;
      x.vp[q] = live ? x.vp[q] : 0u;
      pw[q * kTile + lane] = x.kp[q];
      pw[(NG + q) * kTile + lane] = x.vp[q];
    }
    wave_lds_sync();
    uint32_t top = x.vp[0];
#pragma unroll
    for (int q = 1; q < NG; ++q) top = max(top, x.vp[q]);

    f32x4 s[UPL][RT][NG];
#pragma unroll
    for (int i = 0; i < UPL; ++i)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int q = 0; q < NG; ++q) s[i][rt][q] = f32x4{};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t c = x.k[u][w];
        const f16x8 ka = __builtin_bit_cast(
            f16x8, u32x4{c & LO, c & UP, (c >> 8) & LO, (c >> 8) & UP});
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          s[u / NCL][rt][w / 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              ka, qop[rt][u % NCL][w], s[u / NCL][rt][w / 2], 0, 0, 0);
      }
    }
    // scores, in the row's unit (times f1: log2)
    float y[UPL][RT][4];
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      u32x4 kp[NG];
#pragma unroll
      for (int q = 0; q < NG; ++q)
        kp[q] = *reinterpret_cast<const u32x4*>(pw + q * kTile + (cls + NCL * i) * 16 + 4 * g);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v = 0.f;
#pragma unroll
          for (int q = 0; q < NG; ++q) {
            const float z = pair_zero(kp[q][j]) * qsum[rt][q];
            v = q ? v + z : z;
          }
#pragma unroll
          for (int q = 0; q < NG; ++q)
            v = __builtin_fmaf(pair_step(kp[q][j]), s[i][rt][q][j], v);
          y[i][rt][j] = v;
        }
    }
    // keys that a row does not see (also those past the end)
    if (kTile * t + kTile - 1 > base_pos) {
#pragma unroll
      for (int i = 0; i < UPL; ++i)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (kTile * t + (cls + NCL * i) * 16 + 4 * g + j > qpos[rt]) y[i][rt][j] = -INFINITY;
    }
    float p[UPL][RT][4], ls[RT];
    auto probs = [&](int rt, float r) {
      ls[rt] = 0.f;
#pragma unroll
      for (int i = 0; i < UPL; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[i][rt][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(y[i][rt][j], f1[rt], -r));
          ls[rt] += p[i][rt][j];
        }
    };
    bool past = top > cap;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      probs(rt, ref[rt]);
      past = past || !(ls[rt] <= limit);
    }
    if (__builtin_amdgcn_ballot_w64(past)) {
      // 2^e for the largest step yet: its product below 1, up to 8 allowed
      if (__builtin_amdgcn_ballot_w64(top > cap)) {
        uint32_t w = top;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) w = max(w, (uint32_t)__shfl_xor((int)w, off, 64));
        const int ex = min((int)(w >> 26 & 31u), 30);
        if (cap == 0 || 14 - ex < e) {
          const int old = cap ? e : 14 - ex;
          e = 14 - ex;
          const float f = __builtin_amdgcn_ldexpf(1.f, e - old);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            ref[rt] += (float)(old - e);
            l[rt] *= f;
#pragma unroll
            for (int q = 0; q < NG; ++q) zo[rt][q] *= f;
#pragma unroll
            for (int i = 0; i < NT; ++i) o[rt][i] *= f;
          }
          cap = (uint32_t)min(ex + 3, 30) << 26 | 0x03ffffffu;
          limit = __builtin_amdgcn_ldexpf(4096.f, e);
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < UPL; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) mx = fmaxf(mx, y[i][rt][j]);
        mx = max_x32(max_x16(mx)) * f1[rt] - (float)e;
        const float r = fmaxf(ref[rt], mx);
        const float alpha = r == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref[rt] - r);
        ref[rt] = r;
        l[rt] *= alpha;
#pragma unroll
        for (int q = 0; q < NG; ++q) zo[rt][q] *= alpha;
#pragma unroll
        for (int i = 0; i < NT; ++i) o[rt][i] *= alpha;
        probs(rt, r == -INFINITY ? 0.f : r);   // (a row that has seen no key yet)
      }
    }
    // p step (rounded to float16 for the matrix cores: 2^-12 of each at most, as
    // for 16-bit pools) and the sums over p and p zero
    u32x2 pk[UPL][RT][NG];
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      u32x4 vp[NG];
#pragma unroll
      for (int q = 0; q < NG; ++q)
        vp[q] = *reinterpret_cast<const u32x4*>(pw + (NG + q) * kTile + (cls + NCL * i) * 16 +
                                                4 * g);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          float ps4[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ps4[j] = p[i][rt][j] * pair_step(vp[q][j]);
            // (a key that the row does not see may hold NaN)
            if (kTile * t + kTile - 1 > base_pos && p[i][rt][j] == 0.f) {
              ps4[j] = 0.f;
            } else {
              zo[rt][q] = __builtin_fmaf(p[i][rt][j], pair_zero(vp[q][j]), zo[rt][q]);
            }
          }
          const f16x2 a0{(_Float16)ps4[0], (_Float16)ps4[2]}, a1{(_Float16)ps4[1], (_Float16)ps4[3]};
          pk[i][rt][q] = u32x2{__builtin_bit_cast(uint32_t, a0), __builtin_bit_cast(uint32_t, a1)};
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] += ls[rt];
    // O^T += V^T P^T, two units a product
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int ua = 2 * m, ub = 2 * m + 1;
      u32x4 pb[RT][NG];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          const u32x2 pa = pk[ua / NCL][rt][q], pz = pk[ub / NCL][rt][q];
          const bool ina = NCL == 1 || cls == ua % NCL, inb = NCL == 1 || cls == ub % NCL;
          pb[rt][q] = u32x4{ina ? pa[0] : 0u, ina ? pa[1] : 0u, inb ? pz[0] : 0u,
                            inb ? pz[1] : 0u};
        }
#pragma unroll
      for (int b = 0; b < W; ++b) {
        const uint32_t wa = x.v[ua][b], wb = x.v[ub][b];
        const f16x8 lo = __builtin_bit_cast(
            f16x8, u32x4{wa & LO, (wa >> 8) & LO, wb & LO, (wb >> 8) & LO});
        const f16x8 up = __builtin_bit_cast(
            f16x8, u32x4{wa & UP, (wa >> 8) & UP, wb & UP, (wb >> 8) & UP});
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const f16x8 pv = __builtin_bit_cast(f16x8, pb[rt][b / 2]);
          o[rt][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, pv, o[rt][2 * b], 0, 0, 0);
          o[rt][2 * b + 1] =
              __builtin_amdgcn_mfma_f32_16x16x32_f16(up, pv, o[rt][2 * b + 1], 0, 0, 0);
        }
      }
    }
    // (the next tile's words may overwrite these)
    wave_lds_sync();
  };

  const int end = tile0 + n_tiles;
  int t = tile0 + wave;
  if (t < end) {
    Tile xa, xb;
    load(xa, t, load_id(t));
    int id = load_id(t + kWaves);
    for (;;) {
      load(xb, t + kWaves, id);
      id = load_id(t + 2 * kWaves);
      compute(xa, t);
      t += kWaves;
      if (t >= end) break;
      load(xa, t + kWaves, id);
      id = load_id(t + 2 * kWaves);
      compute(xb, t);
      t += kWaves;
      if (t >= end) break;
    }
  }
  if (__builtin_amdgcn_ballot_w64(worst) && lane == 0) flag(a.status, PKV_STATUS_BAD_PAGE);

  // the wave's rows: sums over its lane groups, codes' powers of two, zeros
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float lr = sum_x32(sum_x16(l[rt]));
    const int row = wave * ROWS + rt * 16 + n;
    if (g == 0) {
      m_lds[row] = ref[rt];
      l_lds[row] = lr;
    }
    float z[NG];
#pragma unroll
    for (int q = 0; q < NG; ++q) z[q] = sum_x32(sum_x16(zo[rt][q]));
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float f = i & 1 ? 0x1p20f : 0x1p24f;
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(o[rt][i][j], f, z[i / 4]);
      *reinterpret_cast<f32x4*>(o_lds + row * OP + 16 * i + 4 * g) = v;
    }
  }
  __syncthreads();

  // merge the waves' (and classes') rows: set k of row r
  constexpr int SETS = kWaves * NCL, CH = D / 4;
  const int64_t part = ((int64_t)slot * a.n_kv + h) * a.part_rows;
  auto store = [&](int r, int c4, f32x4 v, float lr) {
    const int tok = r / G;
    typedef T TV4 __attribute__((ext_vector_type(4)));
    TV4 w;
    const float inv = 1.f / lr;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (T)(v[j] * inv);
    *reinterpret_cast<TV4*>(reinterpret_cast<T*>(a.out) +
                            ((int64_t)(q0 + qs + tok) * Hq + h * G + r % G) * D + 4 * c4) = w;
  };
  const int live_rows = min(OROWS, qn * G);
  for (int i = tid; i < live_rows * CH; i += 64 * kWaves) {
    const int r = i / CH, c4 = i % CH;
    auto at = [&](int k) { return NCL > 1 ? (k / NCL) * ROWS + (k % NCL) * RC + r : k * ROWS + r; };
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < SETS; ++k) m = fmaxf(m, m_lds[at(k)]);
    f32x4 v{};
    float lr = 0.f;
#pragma unroll
    for (int k = 0; k < SETS; ++k) {
      const float mk = m_lds[at(k)];
      const float w = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk - m);
      if (w == 0.f) continue;            // (a set that saw no key holds nothing)
      v += *reinterpret_cast<const f32x4*>(o_lds + at(k) * OP + 4 * c4) * w;
      lr += l_lds[at(k)] * w;
    }
    if (slot < 0) {
      store(r, c4, v, lr);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(
          __builtin_bit_cast(u32x4, v), ws_rsrc(a.part_o + part * D, a.part_rows * D * 4),
          (r * D + 4 * c4) * 4, 0, kSc1);
      if (c4 == 0)
        __builtin_amdgcn_raw_buffer_store_b64(
            __builtin_bit_cast(u32x2, f32x2{m, lr}), ws_rsrc(a.part_ml + part * 2, a.part_rows * 8),
            r * 8, 0, kSc1);
    }
  }
  if (slot < 0) return;

  // Publish: the stores above are performed beyond the XCD's cache (sc1), and
  // every wave waits for its own before the count; the workgroup whose count is
  // the last merges, by loads from there. Counters are zero again afterwards.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const int slot0 = it[6], pieces = it[7];
  int32_t* cnt = a.counters + (int64_t)slot0 * a.n_kv + h;
  if (tid == 0) arrived = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived != pieces - 1) return;
  if (tid == 0) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int i = tid; i < live_rows * CH; i += 64 * kWaves) {
    const int r = i / CH, c4 = i % CH;
    float m = -INFINITY, lr = 0.f;
    f32x4 v{};
    for (int k = 0; k < pieces; ++k) {
      const int64_t pk = ((int64_t)(slot0 + k) * a.n_kv + h) * a.part_rows;
      const f32x2 ml = __builtin_bit_cast(
          f32x2, __builtin_amdgcn_raw_buffer_load_b64(
                     ws_rsrc(a.part_ml + pk * 2, a.part_rows * 8), r * 8, 0, kSc1));
      const f32x4 ov = __builtin_bit_cast(
          f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                     ws_rsrc(a.part_o + pk * D, a.part_rows * D * 4), (r * D + 4 * c4) * 4, 0,
                     kSc1));
      if (ml[0] == -INFINITY) continue;
      const float mn = fmaxf(m, ml[0]);
      const float wa = __builtin_amdgcn_exp2f(m - mn), wb = __builtin_amdgcn_exp2f(ml[0] - mn);
      v = v * wa + ov * wb;
      lr = lr * wa + ml[1] * wb;
      m = mn;
    }
    store(r, c4, v, lr);
  }
}

// ------------------------------------------------------------------- plan ---

static bool fast_4bit(int32_t n_heads, int32_t n_kv, int32_t d, int32_t ps, int32_t dtype) {
  const int32_t units = ps / 16;
  return (dtype == PKV_DTYPE_F16 || dtype == PKV_DTYPE_BF16) && (d == 64 || d == 128) &&
         ps % 16 == 0 && units > 0 && (units & (units - 1)) == 0 && n_heads / n_kv <= 32;
}

static int64_t counter_bytes(int64_t slots, int32_t n_kv) {
  return (slots * n_kv * 4 + 255) / 256 * 256;
}

}  // namespace pkv

using namespace pkv;

extern "C" {

static int plan_4bit(const int32_t* cu_query_lens, const int32_t* kv_indptr, const int32_t* kv_lens,
                  const int32_t* kv_last_page_len, int32_t n_seqs, int32_t n_heads,
                  int32_t n_kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype,
                  int32_t workgroups, int32_t* items, int64_t capacity, int64_t* needed,
                  pkv_4bit* plan) {
  const int rc0 = check_4bit(n_kv_heads, head_dim, page_size);
  if (rc0) return rc0;
  if (n_seqs <= 0 || n_heads <= 0 || n_heads % n_kv_heads || workgroups <= 0)
    return fail(PKV_ERR_INVALID, "n_seqs, n_heads and workgroups must be positive, n_heads a "
                                 "multiple of n_kv_heads");
  if (cu_query_lens[0] != 0 || kv_indptr[0] != 0)
    return fail(PKV_ERR_INVALID, "cu_query_lens and kv_indptr must start at 0");
  plan->n_few = plan->n_wide = plan->few_rows = plan->n_slots = plan->part_rows = 0;
  plan->workspace_bytes = 0;
  *needed = 0;
  const int32_t G = n_heads / n_kv_heads;
  const bool fast = fast_4bit(n_heads, n_kv_heads, head_dim, page_size, dtype);
  int64_t total = 0;      // tiles, over the KV heads
  int32_t few = 0;
  bool wide = false;
  for (int32_t i = 0; i < n_seqs; ++i) {
    const int rc = check_seq_pages(i, kv_indptr[i + 1] - kv_indptr[i], kv_lens[i],
                                   kv_last_page_len[i], page_size);
    if (rc) return rc;
    const int32_t ql = cu_query_lens[i + 1] - cu_query_lens[i];
    if (ql < 1 || ql > kv_lens[i])
      return fail(PKV_ERR_INVALID, "seq %d: query_len=%d outside [1, kv_len=%d]", i, ql,
                  kv_lens[i]);
    if (!fast) continue;
    const int64_t rows = (int64_t)ql * G;
    if (rows <= 16) few = std::max(few, (int32_t)rows);
    else wide = true;
    const int32_t step = rows <= 16 ? ql : std::max(1, 32 / G);
    for (int32_t q = 0; q < ql; q += step)
      total += (kv_lens[i] - ql + std::min(q + step, ql) + kTile - 1) / kTile;
  }
  if (!fast) return PKV_OK;
  plan->few_rows = few == 0 ? 0 : few <= 4 ? 4 : few <= 8 ? 8 : 16;
  plan->part_rows = wide ? 32 : plan->few_rows;
  // A piece: a tile a wave at least, and about as many pieces as workgroups.
  const int64_t piece = std::max<int64_t>(kWaves, (total * n_kv_heads + workgroups - 1) / workgroups);
  struct Piece { int32_t v[kPieceInts]; };
  std::vector<Piece> out[2];
  int32_t slots = 0;
  for (int32_t i = 0; i < n_seqs; ++i) {
    const int32_t ql = cu_query_lens[i + 1] - cu_query_lens[i];
    const int64_t rows = (int64_t)ql * G;
    const int32_t step = rows <= 16 ? ql : std::max(1, 32 / G);
    for (int32_t q = 0; q < ql; q += step) {
      const int32_t qn = std::min(step, ql - q);
      const int32_t tiles = (kv_lens[i] - ql + q + qn + kTile - 1) / kTile;
      // (a remainder below half a piece is shared out among the others)
      const int32_t n = (int32_t)std::max<int64_t>(1, (tiles + piece / 2) / piece);
      const int32_t slot0 = slots;
      if (n > 1) {
        if ((int64_t)slots + n > 0x7fffffff / 64)
          return fail(PKV_ERR_INVALID, "the batch takes too many pieces");
        slots += n;
      }
      int32_t t0 = 0;
      for (int32_t k = 0; k < n; ++k) {
        const int32_t t1 = (int32_t)((int64_t)tiles * (k + 1) / n);
        out[rows > 16].push_back({{i, q, qn, t0, t1 - t0, n > 1 ? slot0 + k : -1, slot0, n}});
        t0 = t1;
      }
    }
  }
  for (auto& v : out)
    std::stable_sort(v.begin(), v.end(), [](const Piece& a, const Piece& b) {
      return a.v[4] > b.v[4];
    });
  *needed = (int64_t)(out[0].size() + out[1].size()) * kPieceInts;
  plan->n_few = (int32_t)out[0].size();
  plan->n_wide = (int32_t)out[1].size();
  plan->n_slots = slots;
  plan->workspace_bytes =
      slots ? counter_bytes(slots, n_kv_heads) +
                  (int64_t)slots * n_kv_heads * plan->part_rows * (head_dim + 2) * 4
            : 0;
  if (*needed > capacity)
    return fail(PKV_ERR_CAPACITY, "plan needs %lld entries, capacity %lld", (long long)*needed,
                (long long)capacity);
  int32_t* at = items;
  for (const auto& v : out)
    for (const Piece& p : v) {
      std::copy(p.v, p.v + kPieceInts, at);
      at += kPieceInts;
    }
  return PKV_OK;
}

int pkv_plan_4bit(const int32_t* cu_query_lens, const int32_t* kv_indptr, const int32_t* kv_lens,
                  const int32_t* kv_last_page_len, int32_t n_seqs, int32_t n_heads,
                  int32_t n_kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype,
                  int32_t workgroups, int32_t* items, int64_t capacity, int64_t* needed,
                  pkv_4bit* plan) {
  if (!cu_query_lens || !kv_indptr || !kv_lens || !kv_last_page_len || !needed || !plan ||
      capacity < 0 || (capacity && !items))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  try {
    return plan_4bit(cu_query_lens, kv_indptr, kv_lens, kv_last_page_len, n_seqs, n_heads,
                     n_kv_heads, head_dim, page_size, dtype, workgroups, items, capacity, needed,
                     plan);
  } catch (const std::exception& e) {
    return fail(PKV_ERR_CAPACITY, "planning failed: %s", e.what());
  }
}

int pkv_attend_4bit(const void* batch, const void* q, void* out, const void* k_pool,
                    const void* v_pool, float scale, void* stream) {
  if (!batch) return fail(PKV_ERR_INVALID, "null pointer argument");
  const pkv_4bit& b = *(const pkv_4bit*)batch;
  const int rc = check_4bit(b.n_kv_heads, b.head_dim, b.page_size);
  if (rc) return rc;
  if (b.n_heads <= 0 || b.n_heads % b.n_kv_heads || b.n_seqs <= 0 || b.n_tokens <= 0 ||
      b.num_blocks < 0 || !elem_bytes(b.dtype))
    return fail(PKV_ERR_INVALID, "the batch's geometry is invalid");
  if (!q || !out || !k_pool || !v_pool || !b.cu_query_lens || !b.kv_indptr || !b.kv_indices ||
      !b.kv_lens)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  hipStream_t s = (hipStream_t)stream;
  if (!fast_4bit(b.n_heads, b.n_kv_heads, b.head_dim, b.page_size, b.dtype)) {
    if (!b.batch_indices) return fail(PKV_ERR_INVALID, "null pointer argument");
    return run_4bit_any(b, q, out, k_pool, v_pool, scale, s);
  }
  if (!b.items || b.n_few + b.n_wide <= 0 || b.n_few < 0 || b.n_wide < 0)
    return fail(PKV_ERR_INVALID, "the batch has no plan");
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool) % 16)
    return fail(PKV_ERR_INVALID, "q, out and the pools have to be aligned to 16 bytes");
  const FourBit f = four_bit(b.n_kv_heads, b.head_dim, b.page_size);
  const int64_t need = b.n_slots ? counter_bytes(b.n_slots, b.n_kv_heads) +
                                       (int64_t)b.n_slots * b.n_kv_heads * b.part_rows *
                                           (b.head_dim + 2) * 4
                                 : 0;
  if (b.workspace_bytes < need || (need && ((uintptr_t)b.workspace % 256 || !b.workspace)))
    return fail(PKV_ERR_INVALID, "workspace of %lld bytes at %p; %lld, aligned to 256, are needed",
                (long long)b.workspace_bytes, b.workspace, (long long)need);
  Attend4 a;
  a.q = q;
  a.out = out;
  a.kpool = (const unsigned char*)k_pool;
  a.vpool = (const unsigned char*)v_pool;
  a.cu_q = b.cu_query_lens;
  a.indptr = b.kv_indptr;
  a.indices = b.kv_indices;
  a.kv_lens = b.kv_lens;
  a.counters = (int32_t*)b.workspace;
  a.part_o = (float*)((char*)b.workspace + counter_bytes(b.n_slots, b.n_kv_heads));
  a.part_ml = a.part_o + (int64_t)b.n_slots * b.n_kv_heads * b.part_rows * b.head_dim;
  a.status = b.status_word;
  a.num_blocks = b.num_blocks;
  a.block = f.block;
  a.n_kv = b.n_kv_heads;
  a.groups = b.n_heads / b.n_kv_heads;
  a.head_bytes = f.head_bytes;
  a.pairs = f.pairs;
  a.shift = __builtin_ctz(b.page_size / 16);
  a.part_rows = b.part_rows;
  a.scale_log2 = scale * kLog2e;
  auto go = [&](auto kernel, const int32_t* items, int32_t n) -> int {
    a.items = items;
    a.n_items = n;
    const int64_t grid = (int64_t)((n + 7) / 8) * 8 * b.n_kv_heads;
    if (grid > 0x7fffffffLL) return fail(PKV_ERR_INVALID, "too many pieces");
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * kWaves), 0, s, a);
    PKV_LAUNCH_CHECK();
    return PKV_OK;
  };
  auto by_rows = [&](auto type, auto dim) -> int {
    typedef decltype(type) T;
    constexpr int D = decltype(dim)::value;
    if (b.n_few) {
      const int rc = b.few_rows == 4   ? go(attend_4bit_kernel<T, D, 1, 4>, b.items, b.n_few)
                     : b.few_rows == 8 ? go(attend_4bit_kernel<T, D, 1, 2>, b.items, b.n_few)
                                       : go(attend_4bit_kernel<T, D, 1, 1>, b.items, b.n_few);
      if (rc) return rc;
    }
    if (b.n_wide)
      return go(attend_4bit_kernel<T, D, 2, 1>, b.items + (int64_t)b.n_few * kPieceInts, b.n_wide);
    return PKV_OK;
  };
  auto by_dim = [&](auto type) -> int {
    return b.head_dim == 64 ? by_rows(type, std::integral_constant<int, 64>{})
                            : by_rows(type, std::integral_constant<int, 128>{});
  };
  return b.dtype == PKV_DTYPE_F16 ? by_dim(_Float16{}) : by_dim(__bf16{});
}

}  // extern "C"
