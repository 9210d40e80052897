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
// 2^e that keeps p step within float16 (p 2^e against the reference). e is a row's
// own and follows the steps of the keys that it sees, those of NaN groups left out:
// what a later token holds leaves an earlier one's weights their bits.
//
// 16 sequences of 20000 to 60000 tokens, head_dim 128 (643 MB), take 113 us: HBM, 5.7
// TB/s. 256 of 1 to 2048, head_dim 64 (40 MB), 13.5: starting, one tile's latency and
// the longest piece. 48 with 2 to 6 new tokens over 2000 to 8000 (282 MB) 77: vector
// work, on 32 rows a piece.
#include <algorithm>
#include <exception>
#include <vector>

#include "attend_fourbit.h"

namespace pkv {

int check_seq_pages(int32_t i, int32_t np, int32_t kv, int32_t last, int32_t ps);
int check_4bit(int32_t n_kv, int32_t d, int32_t ps);
int run_4bit_any(const pkv_4bit& b, const void* q, void* out, const void* k_pool,
                 const void* v_pool, float scale, hipStream_t s);

// Query rows of a piece (few, wide; a sequence of more than kTallFrom may be tall).
constexpr int kFewRows = 16, kWideRows = 32, kTallFrom = 64;
// Pieces of a cut row at most, four waves and one: what the last of them joins.
constexpr int kMostPieces = 128, kMostPieces1 = 32;
// Workgroups a compute unit that pieces are cut for. Few rows, four waves: 2 (one
// sequence of 32750 tokens, head_dim 64: 12.4 us; 1 took 11.9, 4 15.9; 16 of 20000 to
// 60000, head_dim 128: 113, 145 and 115). Wide rows: 2 (48 sequences of 2000 to 8000 with
// 2 to 6 new tokens, head_dim 128: 76.8; 1 took 89.8, 4 78.9).
constexpr int kFewResident = 2, kWideResident = 2;
// From kOneWaveRows rows (x KV heads) a compute unit on, a piece of few rows is one
// wave's, of kOneLeast tiles at least, 16 a compute unit: 256 sequences of 1 to 2048
// tokens (258 on average) take 13.5 us, as four waves' 15.1; pieces from 3 tiles 14.7,
// from 5 and 6 13.7, from 8 15.4. (100 and 500 sequences, and 300 of 100 to 1000: 4, 5, 6
// and 8 within 2%.)
constexpr int kOneResident = 16, kOneLeast = 4, kOneWaveRows = 8;
// Few rows beside wide ones run as wide ones up to kJoin times their tiles: one launch
// with one ramp and tail, for a row of them at least half idle in the matrix cores.
constexpr int kJoin = 4;
// A sequence is tall where kTallAlong tiles x compute units <= work (tiles of all wide
// pieces): a tile takes a tall piece by itself 1.7 us at head_dim 64, a wide one 1.3 us
// / 4 of a compute unit (2.9 and 1.9 / 4 at 128). Measured, 4 query heads each of 8, tall
// and wide: 8 chunks of 512 over 1536 148 and 185 us (head_dim 128: 266 and 320), 16 of
// 512 over 100 72 and 114, 64 of 20 over 300 32 and 42 (128); one of 2000 tokens 58 and
// 47, 8 of 128 over 1000 35 and 31.
constexpr int64_t kTallAlong = 5;

// Floats per wave for a tile's steps, zeros of K, steps and middles of V
// ([4][group][key]).
template <int D> constexpr int kPairFloats = 4 * (D / 64) * kTile;

// Waves a SIMD the kernel is compiled for.
template <int D, int RT> constexpr int kSimdWaves = RT == 2 ? 2 : D == 64 ? 4 : 2;

// WPP: waves of a piece (its team). A workgroup has four waves at least: one-wave
// teams share none but the dispatch (2840 of them began within 0.6 us of each
// other, 2.0 us as workgroups of their own).
template <typename T, int D, int RT, int NCL, int WPP>
__global__ __launch_bounds__(WPP < 4 ? 256 : 64 * WPP, (kSimdWaves<D, RT>))
void attend_4bit_kernel(Attend4 a) {
  constexpr int NG = D / 64;         // groups
  constexpr int W = D / 32;          // words of codes a lane takes of a unit
  constexpr int NT = D / 16;         // output tiles of 16 dims
  constexpr int RC = 16 / NCL;       // rows of a class
  constexpr int PASSES = RT;         // of a tile: 4 / PASSES units each (registers)
  constexpr int UPP = 4 / PASSES;    // units of a pass
  constexpr int UPL = UPP / NCL;     // those whose scores a lane holds
  constexpr int ROWS = RT * 16;      // columns of S^T
  constexpr int OROWS = NCL > 1 ? RC : ROWS;
  constexpr int OP = D + 4;          // floats of a row of the merge's LDS
  constexpr int NTH = 64 * WPP;      // threads of a team
  constexpr int TEAMS = WPP < 4 ? 4 / WPP : 1;
  static_assert(RT == 1 || NCL == 1, "classes are for few rows");
  static_assert(WPP == 1 || TEAMS == 1, "a team is a wave or a workgroup");
  // steps and zeros of a tile; then the merges' sums
  constexpr int PAIR_F = WPP * kPairFloats<D>, RED_F = NTH * 6;
  __shared__ __align__(16) float pair_all[TEAMS][PAIR_F > RED_F ? PAIR_F : RED_F];
  __shared__ __align__(16) float o_all[TEAMS][WPP * ROWS * OP];
  __shared__ float m_all[TEAMS][WPP * ROWS], l_all[TEAMS][WPP * ROWS];
  __shared__ int arrived;

  const int wave_of_block = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = WPP == 1 ? wave_of_block : 0, wave = WPP == 1 ? 0 : wave_of_block;
  const int tid = WPP == 1 ? threadIdx.x & 63 : threadIdx.x;
  float* const pair_lds = pair_all[team];
  float* const o_lds = o_all[team];
  float* const m_lds = m_all[team];
  float* const l_lds = l_all[team];
  auto team_sync = [&]() {
    if constexpr (WPP == 1) wave_lds_sync();
    else __syncthreads();
  };

  // Eight XCDs take workgroups in turn; a piece's heads go to one of them, where
  // they share the lines that hold steps and zeros of two heads.
  const int x = blockIdx.x & 7, y = (blockIdx.x >> 3) * TEAMS + team;
  const int item = (y / a.n_kv) * 8 + x, h = y % a.n_kv;
  if (item >= a.n_items) return;
  const int32_t* it = a.items + (int64_t)item * kPieceInts;
  const int q0 = it[0], qn = it[1], base_pos = it[2], kv_len = it[3], pbase = it[4],
            n_pages = it[5], tile0 = it[6], n_tiles = it[7], slot = it[8];
  const int G = a.groups, Hq = a.n_kv * G;
  const int lane = tid & 63, g = lane >> 4, n = lane & 15;
  const int cls = NCL > 1 ? n / RC : 0;

  // The tile being computed and the next one share registers: K's are loaded again
  // once its products are through, V's likewise, so that a tile's K is on its way
  // during the softmax and V's products of the one before, its V during the rest.
  uint32_t kc[4][W], vc[4][W];       // codes
  uint32_t kw[NG], vw[NG];           // the words of key `lane`
  const int shift = a.shift, mask = (1 << shift) - 1;    // units of a page
  auto load_id = [&](int t) {      // the page of lane group g's unit of tile t
    return a.indices[pbase + min((4 * t + g) >> shift, n_pages - 1)];
  };
  constexpr uint32_t unit_bytes = 8 * D;
  const uint32_t k_off = h * a.head_bytes + n * (D / 2) + g * (D / 8);
  const uint32_t v_off = h * a.head_bytes + lane * (D / 8);
  const int ps = 16 << shift;
  typedef uint32_t Words __attribute__((ext_vector_type(W)));
  int64_t at[4];                     // where the units of the tile being loaded begin
  auto codes = [&](uint32_t (&to)[4][W], const unsigned char* pool, uint32_t off) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      // (a scalar base and a lane's 32-bit offset)
      const Words x = __builtin_nontemporal_load(reinterpret_cast<const Words*>(pool + at[u] + off));
#pragma unroll
      for (int w = 0; w < W; ++w) to[u][w] = x[w];
    }
  };
  auto load_k = [&](int t, int id) {
    const int ok = (uint64_t)(int64_t)id < (uint64_t)a.num_blocks ? id : 0;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      at[u] = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(ok, 16 * u) * (uint32_t)a.block +
              ((4 * t + u) & mask) * unit_bytes;
    const uint64_t mine = (uint64_t)(uint32_t)ok * (uint32_t)a.block +
                          (uint32_t)(a.pairs + ((h * NG) * ps + ((4 * t + g) & mask) * 16 + n) * 4);
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      kw[q] = __builtin_nontemporal_load(
          reinterpret_cast<const uint32_t*>(a.kpool + mine + q * ps * 4));
      vw[q] = __builtin_nontemporal_load(
          reinterpret_cast<const uint32_t*>(a.vpool + mine + q * ps * 4));
    }
    codes(kc, a.kpool, k_off);
  };
  auto load_v = [&]() { codes(vc, a.vpool, v_off); };   // of load_k's tile

  // the first tile goes out before the queries are read
  const int end = tile0 + n_tiles;
  int t = tile0 + wave;
  int id = 0, id_next = 0;           // of tiles t, t + WPP
  if (t < end) {
    const int32_t* first = it + 12 + 4 * wave;         // (its pages came with the piece)
    id = g == 0 ? first[0] : g == 1 ? first[1] : g == 2 ? first[2] : first[3];
    load_k(t, id);
    load_v();
    id_next = load_id(t + WPP);
  }

  auto token_of = [&](int r) { return (int)((uint32_t)r * a.per_group >> 16); };   // r / G
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
    const int tok = token_of(r);
    const bool valid = tok < qn;
    const int head = valid ? r - tok * G : 0;
    qpos[rt] = base_pos + (valid ? tok : qn - 1);
    typedef T TV __attribute__((ext_vector_type(8)));
    const T* row = reinterpret_cast<const T*>(a.q) +
                   ((int64_t)(q0 + (valid ? tok : 0)) * Hq + h * G + head) * D + 16 * g;
    float v[2 * NG][8], mx = 0.f;
#pragma unroll
    for (int w = 0; w < 2 * NG; ++w) {
      const TV t = *reinterpret_cast<const TV*>(row + (w >> 1) * 64 + (w & 1) * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[w][i] = Elem<T>::to_f(t[i]);
        mx = fmaxf(mx, __builtin_fabsf(v[w][i]));
      }
    }
    mx = max_x32(max_x16(mx));
    const bool scaled = mx > 0.f && mx < INFINITY;
    const int k = scaled ? 11 - __builtin_amdgcn_frexp_expf(mx) : 0;
    const uint32_t turn = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    // (a scale of 0: small enough to change nothing, and no 0 x inf at masks)
    f1[rt] = __builtin_amdgcn_ldexpf(__builtin_fabsf(a.scale_log2), 24 - k);
    f1[rt] = f1[rt] < 0x1p-120f ? 0x1p-120f : f1[rt];
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      float sum = 0.f;
#pragma unroll
      for (int w = 2 * q; w < 2 * q + 2; ++w) {
        u32x4 op;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                 // elements i and i + 4
          const int down = i & 1 ? 4 : 0;             // their codes lie four bits up
          const f16x2 two{(_Float16)__builtin_amdgcn_ldexpf(v[w][i], k - down),
                          (_Float16)__builtin_amdgcn_ldexpf(v[w][i + 4], k - down)};
          const f16x2 turned = __builtin_bit_cast(f16x2, __builtin_bit_cast(uint32_t, two) ^ turn);
          sum = __builtin_fmaf((float)turned[0], (float)(1 << down), sum);
          sum = __builtin_fmaf((float)turned[1], (float)(1 << down), sum);
          op[i] = __builtin_bit_cast(uint32_t, turned);
        }
#pragma unroll
        for (int c = 0; c < NCL; ++c)
          qop[rt][c][w] = __builtin_bit_cast(
              f16x8, valid && (NCL == 1 || c == cls) ? op : u32x4{0u, 0u, 0u, 0u});
      }
      sum = sum_x32(sum_x16(sum)) * 0x1p-24f;
      qsum[rt][q] = valid ? sum : 0.f;
    }
  }

  f32x4 o[RT][NT], pr[RT][NG];
  float ref[RT], l[RT], zo[RT][NG];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int i = 0; i < NT; ++i) o[rt][i] = f32x4{};
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      zo[rt][q] = 0.f;
      pr[rt][q] = f32x4{};
    }
    ref[rt] = -INFINITY;
    l[rt] = 0.f;
  }
  // of each row: the largest step (a word's) that 2^e allows, e, 2^12 2^e. (The same
  // in all rows, and in scalar registers, until a tile is seen in part.)
  uint32_t cap[RT];
  int e[RT];
  float limit[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    cap[rt] = 0;
    e[rt] = 0;
    limit[rt] = 4096.f;
  }
  uint32_t worst = 0;                // any page id out of range
  float* const pw = pair_lds + wave * kPairFloats<D>;
  const uint32_t LO = 0x000f000fu, UP = 0x00f000f0u;

  // Tile t. PART: some row does not see all of its keys; MORE: load the next one.
  auto compute = [&](auto part, auto more) {
    constexpr bool PART = decltype(part)::value, MORE = decltype(more)::value;
    // steps and zeros; none for keys past the end and for pages out of range,
    // which read as zeros
    const bool bad = (uint64_t)(int64_t)id >= (uint64_t)a.num_blocks;
    const bool live = (!PART || kTile * t + lane < kv_len) && !bad;
    worst |= bad;
    uint32_t top = 0;                // the key's largest step, then that of keys up to it
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const uint32_t kp = live ? kw[q] : 0u, vp = live ? vw[q] : 0u;
      top = max(top, vp < kNoStep ? vp : 0u);
      const float step = pair_step(vp);
      pw[q * kTile + lane] = pair_step(kp);
      pw[(NG + q) * kTile + lane] = pair_zero(kp);
      pw[(2 * NG + q) * kTile + lane] = step;
      pw[(3 * NG + q) * kTile + lane] = __builtin_fmaf(7.5f, step, pair_zero(vp));
    }
    wave_lds_sync();
    uint32_t seen[RT];               // the largest step among a row's keys of the tile
    if constexpr (PART) {
      top = scan_max(top);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int last = qpos[rt] - kTile * t;
        const uint32_t w = (uint32_t)__shfl((int)top, min(max(last, 0), kTile - 1), 64);
        seen[rt] = last < 0 ? 0u : w;
      }
    }

    auto pairs = [&](int kind, int q, int u) {   // of the lane's four keys of unit u
      return *reinterpret_cast<const f32x4*>(pw + (kind * NG + q) * kTile + (cls + u) * 16 + 4 * g);
    };
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
    const int u0 = ps * UPP;         // the pass's first unit
    f32x4 s[UPL][RT][NG];
#pragma unroll
    for (int i = 0; i < UPL; ++i)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int q = 0; q < NG; ++q) s[i][rt][q] = f32x4{};
#pragma unroll
    for (int u = 0; u < UPP; ++u) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t c = kc[u0 + u][w];
        const f16x8 ka = __builtin_bit_cast(
            f16x8, u32x4{c & LO, c & UP, (c >> 8) & LO, (c >> 8) & UP});
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          s[u / NCL][rt][w / 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              ka, qop[rt][u % NCL][w], s[u / NCL][rt][w / 2], 0, 0, 0);
      }
    }
    // (Nothing moves across the phases: the compiler would unpack all of a tile's
    // codes ahead of their products, and run out of registers.)
    __builtin_amdgcn_sched_barrier(0);
    if (ps == PASSES - 1) {
      if constexpr (MORE) load_k(t + WPP, id_next);
    }
    auto unseen = [&](int rt, int i, int j) {    // key j of the lane's unit i of the pass
      return kTile * t + (u0 + cls + NCL * i) * 16 + 4 * g + j > qpos[rt];
    };
    // scores, in the row's unit (times f1: log2)
    float y[UPL][RT][4];
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
      asm volatile("" ::: "memory");   // (reads no earlier: registers)
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        const f32x4 step = pairs(0, q, u0 + NCL * i), zero = pairs(1, q, u0 + NCL * i);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float z = q ? __builtin_fmaf(zero[j], qsum[rt][q], y[i][rt][j])
                              : zero[j] * qsum[rt][q];
            y[i][rt][j] = __builtin_fmaf(step[j], s[i][rt][q][j], z);
          }
      }
    }
    if constexpr (PART) {            // (also keys past the end)
#pragma unroll
      for (int i = 0; i < UPL; ++i)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (unseen(rt, i, j)) y[i][rt][j] = -INFINITY;
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
    bool past = false, more_step = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (ps == 0) more_step = more_step || (PART ? seen[rt] : top) > cap[rt];
      probs(rt, ref[rt]);
      past = past || !(ls[rt] <= limit[rt]);
    }
    if (__builtin_amdgcn_ballot_w64(past || more_step)) {
      // 2^e for the largest step yet: its product below 1, up to 8 allowed
      if (ps == 0 && __builtin_amdgcn_ballot_w64(more_step)) {
        if constexpr (!PART) {
          const uint32_t w = (uint32_t)__builtin_amdgcn_readlane((int)scan_max(top), 63);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) seen[rt] = w;
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const int ex = (int)(seen[rt] >> 26);
          const bool moves = seen[rt] > cap[rt];
          const int now = moves ? 14 - ex : e[rt];
          const float f = __builtin_amdgcn_ldexpf(1.f, now - e[rt]);
          ref[rt] += (float)(e[rt] - now);
          l[rt] *= f;
#pragma unroll
          for (int q = 0; q < NG; ++q) {
            zo[rt][q] *= f;
            pr[rt][q] *= f;
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) o[rt][i] *= f;
          e[rt] = now;
          if (moves) cap[rt] = (uint32_t)min(ex + 3, 30) << 26 | 0x03ffffffu;
          limit[rt] = __builtin_amdgcn_ldexpf(4096.f, now);
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < UPL; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) mx = fmaxf(mx, y[i][rt][j]);
        mx = max_x32(max_x16(mx)) * f1[rt] - (float)e[rt];
        const float r = fmaxf(ref[rt], mx);
        const float alpha = r == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref[rt] - r);
        ref[rt] = r;
        l[rt] *= alpha;
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          zo[rt][q] *= alpha;
          pr[rt][q] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) o[rt][i] *= alpha;
        probs(rt, r == -INFINITY ? 0.f : r);   // (a row that has seen no key yet)
      }
    }
    // p step, rounded to float16 for the matrix cores, and the sum over p (zero +
    // 7.5 step). With the sum of the rounded ones (a product with ones) taken off
    // 7.5 times at the end, a rounding's error enters with c - 7.5, the value about
    // the group's middle, as it would with 16-bit values; with c alone the outputs
    // were off twice as far.
    u32x2 pk[UPL][RT][NG];
#pragma unroll
    for (int i = 0; i < UPL; ++i)
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        asm volatile("" ::: "memory");
        const f32x4 step = pairs(2, q, u0 + NCL * i), mid = pairs(3, q, u0 + NCL * i);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float w[4], z = zo[rt][q];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float pj = p[i][rt][j];
            // (a key that the row does not see may hold NaN; one that it sees counts
            // however small its weight)
            const bool none = PART && unseen(rt, i, j);
            w[j] = none ? 0.f : pj * step[j];
            z = none ? z : __builtin_fmaf(pj, mid[j], z);
          }
          zo[rt][q] = z;
          const f16x2 a0{(_Float16)w[0], (_Float16)w[2]}, a1{(_Float16)w[1], (_Float16)w[3]};
          pk[i][rt][q] = u32x2{__builtin_bit_cast(uint32_t, a0), __builtin_bit_cast(uint32_t, a1)};
        }
      }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] += ls[rt];
    // O^T += V^T P^T, two units a product
    const f16x8 ones = __builtin_bit_cast(
        f16x8, u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u});
#pragma unroll
    for (int m = 0; m < UPP / 2; ++m) {
      __builtin_amdgcn_sched_barrier(0);
      const int ua = 2 * m, ub = 2 * m + 1;      // of the pass
      f16x8 pb[RT][NG];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          const u32x2 pa = pk[ua / NCL][rt][q], pz = pk[ub / NCL][rt][q];
          const bool ina = NCL == 1 || cls == ua % NCL, inb = NCL == 1 || cls == ub % NCL;
          pb[rt][q] = __builtin_bit_cast(
              f16x8, u32x4{ina ? pa[0] : 0u, ina ? pa[1] : 0u, inb ? pz[0] : 0u,
                           inb ? pz[1] : 0u});
          pr[rt][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[rt][q], pr[rt][q], 0, 0, 0);
        }
#pragma unroll
      for (int b = 0; b < W; ++b) {
        const uint32_t wa = vc[u0 + ua][b], wb = vc[u0 + ub][b];
        const f16x8 lo = __builtin_bit_cast(
            f16x8, u32x4{wa & LO, (wa >> 8) & LO, wb & LO, (wb >> 8) & LO});
        const f16x8 up = __builtin_bit_cast(
            f16x8, u32x4{wa & UP, (wa >> 8) & UP, wb & UP, (wb >> 8) & UP});
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          o[rt][2 * b] =
              __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, pb[rt][b / 2], o[rt][2 * b], 0, 0, 0);
          o[rt][2 * b + 1] =
              __builtin_amdgcn_mfma_f32_16x16x32_f16(up, pb[rt][b / 2], o[rt][2 * b + 1], 0, 0, 0);
        }
      }
    }
    }
    t += WPP;
    if constexpr (MORE) {
      load_v();
      id = id_next;
      id_next = load_id(t + WPP);
    }
    wave_lds_sync();                 // (the next tile's words overwrite this one's)
  };
  // Whole tiles, then those that some row sees in part, the piece's last ones. (Two
  // loops: with both kinds in one the compiler kept twice the registers.)
  const int whole = min(end, (base_pos + 1) / kTile);
  while (t < whole) compute(std::false_type{}, std::true_type{});
  while (t < end) {
    compute(std::true_type{}, std::false_type{});
    if (t < end) {
      id = id_next;
      load_k(t, id);
      load_v();
      id_next = load_id(t + WPP);
    }
  }
  if (__builtin_amdgcn_ballot_w64(worst) && lane == 0) flag(a.status, PKV_STATUS_BAD_PAGE);

  // the wave's rows: sums over its lane groups, codes' powers of two, middles
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
    for (int q = 0; q < NG; ++q)
      z[q] = __builtin_fmaf(-7.5f, pr[rt][q][0], sum_x32(sum_x16(zo[rt][q])));
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float f = i & 1 ? 0x1p20f : 0x1p24f;
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __builtin_fmaf(o[rt][i][j], f, z[i / 4]);
      *reinterpret_cast<f32x4*>(o_lds + row * OP + 16 * i + 4 * g) = v;
    }
  }
  team_sync();

  // merge the waves' (and classes') rows: set k of row r
  constexpr int SETS = WPP * NCL, CH = D / 4;
  const int64_t part = ((int64_t)slot * a.n_kv + h) * a.part_rows;
  auto store = [&](int r, int c4, f32x4 v, float lr) {
    const int tok = token_of(r);
    typedef T TV4 __attribute__((ext_vector_type(4)));
    TV4 w;
    const float inv = 1.f / lr;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (T)(v[j] * inv);
    *reinterpret_cast<TV4*>(reinterpret_cast<T*>(a.out) +
                            ((int64_t)(q0 + tok) * Hq + h * G + r - tok * G) * D + 4 * c4) = w;
  };
  const int live_rows = min(OROWS, qn * G);
  for (int i = tid; i < live_rows * CH; i += NTH) {
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
      // (a set that saw no key holds zeros)
      const float w = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk - m);
      v += *reinterpret_cast<const f32x4*>(o_lds + at(k) * OP + 4 * c4) * w;
      lr = __builtin_fmaf(l_lds[at(k)], w, lr);
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
  // every wave waits for its own before the count; the team whose count is the
  // last merges, by loads from there. Counters are zero again afterwards.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const int slot0 = it[9], pieces = it[10];
  int32_t* cnt = a.counters + ((int64_t)it[11] * a.n_kv + h) * a.count_step;
  int count = 0;
  if constexpr (WPP == 1) {
    if (lane == 0)
      count = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    count = __builtin_amdgcn_readfirstlane(count);
  } else {
    __syncthreads();
    if (tid == 0)
      arrived = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    count = arrived;
  }
  if (count != pieces - 1) return;
  if (tid == 0) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // A thread per (row, 4 dims), or several, each some of the pieces, where there
  // are fewer; eight pieces' loads are in flight together (none past the last).
  const int apart = a.n_kv * a.part_rows;   // rows between two pieces' of this head
  const int64_t row0 = ((int64_t)slot0 * a.n_kv + h) * a.part_rows;
  const int reach = (pieces - 1) * apart + live_rows;
  const __amdgpu_buffer_rsrc_t mls = ws_rsrc(a.part_ml + row0 * 2, reach * 8);
  const __amdgpu_buffer_rsrc_t os = ws_rsrc(a.part_o + row0 * D, reach * D * 4);
  const int units = live_rows * CH, share = units >= NTH ? 1 : NTH / units;
  for (int i0 = 0; i0 < units; i0 += NTH) {
    const int i = share > 1 ? tid % units : i0 + tid;
    const int first = share > 1 ? tid / units : 0;
    const int r = i / CH, c4 = i % CH;
    const bool mine = i < units && first < share;
    f32x4 v{};
    float m = -INFINITY, lr = 0.f;
    for (int k0 = first; k0 < pieces; k0 += 8 * share) {
      f32x2 ml[8];
      f32x4 ov[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = k0 + j * share;
        const int at = mine && k < pieces ? k * apart + r : reach;
        ml[j] = __builtin_bit_cast(f32x2,
                                   __builtin_amdgcn_raw_buffer_load_b64(mls, at * 8, 0, kSc1));
        ov[j] = __builtin_bit_cast(
            f32x4, __builtin_amdgcn_raw_buffer_load_b128(os, (at * D + 4 * c4) * 4, 0, kSc1));
      }
      float mn = m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (k0 + j * share >= pieces) ml[j][0] = -INFINITY;
        mn = fmaxf(mn, ml[j][0]);
      }
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      v *= f;
      lr *= f;
      m = mn;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = ml[j][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[j][0] - m);
        v += ov[j] * w;
        lr = __builtin_fmaf(ml[j][1], w, lr);
      }
    }
    if (share > 1) {
      f32x4* const red = reinterpret_cast<f32x4*>(pair_lds);
      f32x2* const red2 = reinterpret_cast<f32x2*>(red + NTH);
      red[tid] = v;
      red2[tid] = f32x2{m, lr};
      team_sync();
      if (first == 0) {
        for (int k = 1; k < share; ++k) {
          const f32x2 other = red2[tid + k * units];
          const float mn = fmaxf(m, other[0]);
          // (at -inf: no key, and zeros, or NaN scores alone, and NaN)
          const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
          const float w = other[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(other[0] - mn);
          v = v * f + red[tid + k * units] * w;
          lr = lr * f + other[1] * w;
          m = mn;
        }
        store(r, c4, v, lr);
      }
    } else if (mine) {
      store(r, c4, v, lr);
    }
  }
}

// ------------------------------------------------------------------- plan ---

// (KV heads: 128 pieces' parts of 32 rows lie within 2^31 bytes of each other)
static bool fast_4bit(int32_t n_heads, int32_t n_kv, int32_t d, int32_t ps, int32_t dtype) {
  const int32_t units = ps / 16;
  return (dtype == PKV_DTYPE_F16 || dtype == PKV_DTYPE_BF16) && (d == 64 || d == 128) &&
         ps % 16 == 0 && units > 0 && (units & (units - 1)) == 0 && n_heads / n_kv <= 32 &&
         n_kv <= 256;
}

// Arrival counters lie 128 bytes apart where they are few and their pieces may be
// many: counts of one line are taken one after another, 10 ns each.
static int32_t count_step(int64_t counters) { return counters <= 4096 ? 32 : 1; }
static int64_t counter_bytes(int64_t cuts, int32_t n_kv) {
  const int64_t n = cuts * n_kv;
  return (n * count_step(n) * 4 + 255) / 256 * 256;
}

}  // namespace pkv

using namespace pkv;

extern "C" {

static int plan_4bit(const int32_t* cu_query_lens, const int32_t* kv_indptr,
                     const int32_t* kv_indices, const int32_t* kv_lens,
                     const int32_t* kv_last_page_len, int32_t n_seqs, int32_t n_heads,
                     int32_t n_kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype,
                     int32_t compute_units, int32_t* items, int64_t capacity, int64_t* needed,
                     pkv_4bit* plan) {
  const int rc0 = check_4bit(n_kv_heads, head_dim, page_size);
  if (rc0) return rc0;
  if (n_seqs <= 0 || n_heads <= 0 || n_heads % n_kv_heads || compute_units <= 0)
    return fail(PKV_ERR_INVALID, "n_seqs, n_heads and compute_units must be positive, n_heads a "
                                 "multiple of n_kv_heads");
  if (cu_query_lens[0] != 0 || kv_indptr[0] != 0)
    return fail(PKV_ERR_INVALID, "cu_query_lens and kv_indptr must start at 0");
  plan->n_few = plan->n_wide = plan->n_tall = plan->few_rows = plan->n_slots = plan->part_rows = 0;
  plan->few_waves = plan->n_cuts = 0;
  plan->workspace_bytes = 0;
  *needed = 0;
  const int32_t G = n_heads / n_kv_heads;
  const bool fast = fast_4bit(n_heads, n_kv_heads, head_dim, page_size, dtype);
  struct Row { int32_t seq, q, n, tiles; };      // n tokens of a sequence from its q-th
  std::vector<Row> rows[3];                       // few, wide, tall
  std::vector<int32_t> many;                      // wide or tall sequences
  int64_t tiles[2] = {0, 0}, work = 0;
  int32_t few = 0;
  // Sequence i's rows in parts of a kind; their tiles.
  auto part = [&](int32_t i, int kind, bool keep) {
    const int32_t kv = kv_lens[i], ql = cu_query_lens[i + 1] - cu_query_lens[i];
    const int32_t step = kind == 0 ? ql : std::max(1, (kind == 1 ? kWideRows : kTallRows) / G);
    int64_t sum = 0;
    for (int32_t q = 0; q < ql; q += step) {
      const int32_t n = std::min(step, ql - q);
      const int32_t nt = (kv - ql + q + n + kTile - 1) / kTile;
      if (keep) rows[kind].push_back({i, q, n, nt});
      sum += nt;
    }
    if (keep && kind < 2) tiles[kind] += sum;
    return sum;
  };
  for (int32_t i = 0; i < n_seqs; ++i) {
    const int32_t kv = kv_lens[i], ql = cu_query_lens[i + 1] - cu_query_lens[i];
    // (keys are counted in whole tiles, here and in the kernels)
    if (kv > 0x7fffffff - 2 * kTile)
      return fail(PKV_ERR_INVALID, "seq %d: kv_len=%d is above 2^31 - 129", i, kv);
    const int rc = check_seq_pages(i, kv_indptr[i + 1] - kv_indptr[i], kv, kv_last_page_len[i],
                                   page_size);
    if (rc) return rc;
    if (ql < 1 || ql > kv)
      return fail(PKV_ERR_INVALID, "seq %d: query_len=%d outside [1, kv_len=%d]", i, ql, kv);
    if (!fast) continue;
    const int64_t qr = (int64_t)ql * G;
    if (qr > kTallFrom) {
      many.push_back(i);
      work += part(i, 1, false) * n_kv_heads;
      continue;
    }
    const int kind = qr <= kFewRows ? 0 : 1;
    if (kind == 0) few = std::max(few, ql * G);
    part(i, kind, true);
  }
  // A tall piece runs along all its keys by itself, so a sequence is tall only where
  // its tiles one after the other take no longer than all of the work does, shared
  // out as wide pieces.
  for (const int32_t i : many) {
    const int64_t along = (kv_lens[i] + kTile - 1) / kTile;
    part(i, kTallAlong * along * compute_units <= work ? 2 : 1, true);
  }
  if (!fast) return PKV_OK;
  // Beside wide rows few rows run as wide ones do, unless theirs are most tiles: one
  // launch, with one ramp and one tail.
  if (!rows[1].empty() && tiles[0] <= kJoin * tiles[1]) {
    rows[1].insert(rows[1].end(), rows[0].begin(), rows[0].end());
    rows[0].clear();
    few = 0;
  }
  plan->few_rows = few == 0 ? 0 : few <= 4 ? 4 : few <= 8 ? 8 : 16;
  plan->part_rows = !rows[1].empty() ? kWideRows : plan->few_rows;
  // Many short rows take a wave each, the others four.
  const bool one = (int64_t)rows[0].size() * n_kv_heads >= kOneWaveRows * (int64_t)compute_units;
  plan->few_waves = few ? (one ? 1 : 4) : 0;
  struct Piece { int32_t v[kPieceInts]; };
  std::vector<Piece> out[3];
  const int32_t units = page_size / 16;      // of a page
  int32_t slots = 0, cuts = 0;
  for (int wide = 0; wide < 3; ++wide) {
    // The shortest piece (a tile a wave at least) with which all of them are
    // resident at once: none waits for another to end.
    const bool alone = !wide && one;
    const int64_t resident =
        (int64_t)compute_units * (wide ? kWideResident : alone ? kOneResident : kFewResident);
    const int64_t most = wide == 2 ? 1 : alone ? kMostPieces1 : kMostPieces;
    auto pieces = [&](const Row& r, int64_t piece) {
      return std::min<int64_t>(most, (r.tiles + piece - 1) / piece);
    };
    auto fits = [&](int64_t piece) {
      int64_t n = 0;
      for (const Row& r : rows[wide]) n += pieces(r, piece);
      return n * n_kv_heads <= resident;
    };
    int64_t lo = alone ? kOneLeast : 4, hi = lo;
    for (const Row& r : rows[wide]) hi = std::max<int64_t>(hi, r.tiles);
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (fits(mid)) hi = mid;
      else lo = mid + 1;
    }
    for (const Row& r : rows[wide]) {
      const int32_t i = r.seq, q = r.q, qn = r.n, nt = r.tiles;
      const int32_t ql = cu_query_lens[i + 1] - cu_query_lens[i];
      const int32_t n = (int32_t)pieces(r, lo);
      const int32_t slot0 = slots;
      if (n > 1) {
        if (slots > 0x7fffffff / 64 - n)
          return fail(PKV_ERR_INVALID, "the batch takes too many pieces");
        slots += n;
        ++cuts;
      }
      int32_t t0 = 0;
      for (int32_t k = 0; k < n; ++k) {
        const int32_t t1 = (int32_t)((int64_t)nt * (k + 1) / n);
        Piece p{{cu_query_lens[i] + q, qn, kv_lens[i] - ql + q, kv_lens[i], kv_indptr[i],
                 kv_indptr[i + 1] - kv_indptr[i], t0, t1 - t0, n > 1 ? slot0 + k : -1, slot0, n,
                 cuts - 1}};
        for (int32_t u = 0; u < 16; ++u)
          p.v[12 + u] = kv_indices[kv_indptr[i] + std::min((4 * t0 + u) / units, p.v[5] - 1)];
        out[wide].push_back(p);
        t0 = t1;
      }
    }
  }
  for (auto& v : out)
    std::stable_sort(v.begin(), v.end(), [](const Piece& a, const Piece& b) {
      return a.v[7] > b.v[7];
    });
  *needed = (int64_t)(out[0].size() + out[1].size() + out[2].size()) * kPieceInts;
  plan->n_few = (int32_t)out[0].size();
  plan->n_wide = (int32_t)out[1].size();
  plan->n_tall = (int32_t)out[2].size();
  plan->n_slots = slots;
  plan->n_cuts = cuts;
  plan->workspace_bytes =
      slots ? counter_bytes(cuts, n_kv_heads) +
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

int pkv_plan_4bit(const int32_t* cu_query_lens, const int32_t* kv_indptr,
                  const int32_t* kv_indices, const int32_t* kv_lens,
                  const int32_t* kv_last_page_len, int32_t n_seqs, int32_t n_heads,
                  int32_t n_kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype,
                  int32_t compute_units, int32_t* items, int64_t capacity, int64_t* needed,
                  pkv_4bit* plan) {
  if (!cu_query_lens || !kv_indptr || !kv_indices || !kv_lens || !kv_last_page_len || !needed || !plan ||
      capacity < 0 || (capacity && !items))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  try {
    return plan_4bit(cu_query_lens, kv_indptr, kv_indices, kv_lens, kv_last_page_len, n_seqs,
                     n_heads, n_kv_heads, head_dim, page_size, dtype, compute_units, items, capacity, needed,
                     plan);
  } catch (const std::exception& e) {
    return fail(PKV_ERR_CAPACITY, "planning failed: %s", e.what());
  }
}

int64_t pkv_counter_bytes_4bit(int32_t n_cuts, int32_t n_kv_heads) {
  return n_cuts > 0 && n_kv_heads > 0 ? counter_bytes(n_cuts, n_kv_heads) : 0;
}

int pkv_attend_4bit(const void* batch, const void* q, void* out, const void* k_pool,
                    const void* v_pool, float scale, void* stream) {
  if (!batch) return fail(PKV_ERR_INVALID, "null pointer argument");
  const pkv_4bit& b = *(const pkv_4bit*)batch;
  const int rc = check_4bit(b.n_kv_heads, b.head_dim, b.page_size);
  if (rc) return rc;
  if (b.n_heads <= 0 || b.n_heads % b.n_kv_heads || b.n_seqs <= 0 || b.n_tokens <= 0 ||
      b.num_blocks <= 0 || !elem_bytes(b.dtype))
    return fail(PKV_ERR_INVALID, "the batch's geometry is invalid");
  if (!q || !out || !k_pool || !v_pool || !b.cu_query_lens || !b.kv_indptr || !b.kv_indices ||
      !b.kv_lens)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  hipStream_t s = (hipStream_t)stream;
  if (!fast_4bit(b.n_heads, b.n_kv_heads, b.head_dim, b.page_size, b.dtype)) {
    if (!b.batch_indices) return fail(PKV_ERR_INVALID, "null pointer argument");
    return run_4bit_any(b, q, out, k_pool, v_pool, scale, s);
  }
  if (!b.items || b.n_few < 0 || b.n_wide < 0 || b.n_tall < 0 ||
      (int64_t)b.n_few + b.n_wide + b.n_tall <= 0)
    return fail(PKV_ERR_INVALID, "the batch has no plan");
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool) % 16)
    return fail(PKV_ERR_INVALID, "q, out and the pools have to be aligned to 16 bytes");
  const FourBit f = four_bit(b.n_kv_heads, b.head_dim, b.page_size);
  const int64_t need = b.n_slots ? counter_bytes(b.n_cuts, b.n_kv_heads) +
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
  a.indices = b.kv_indices;
  a.counters = (int32_t*)b.workspace;
  a.part_o = (float*)((char*)b.workspace + counter_bytes(b.n_cuts, b.n_kv_heads));
  a.count_step = count_step((int64_t)b.n_cuts * b.n_kv_heads);
  a.part_ml = a.part_o + (int64_t)b.n_slots * b.n_kv_heads * b.part_rows * b.head_dim;
  a.status = b.status_word;
  a.num_blocks = b.num_blocks;
  a.block = f.block;
  a.n_kv = b.n_kv_heads;
  a.groups = b.n_heads / b.n_kv_heads;
  a.per_group = (65536u + a.groups - 1) / a.groups;
  a.head_bytes = f.head_bytes;
  a.pairs = f.pairs;
  a.shift = __builtin_ctz(b.page_size / 16);
  a.part_rows = b.part_rows;
  a.scale_log2 = scale * kLog2e;
  auto go = [&](auto kernel, const int32_t* items, int32_t n, int waves) -> int {
    a.items = items;
    a.n_items = n;
    // (of each XCD: its pieces' heads, four to a workgroup where a wave takes one)
    const int64_t per_xcd = (int64_t)((n + 7) / 8) * b.n_kv_heads;
    const int64_t grid = (waves == 1 ? (per_xcd + 3) / 4 : per_xcd) * 8;
    if (!launchable(grid, 256)) return fail(PKV_ERR_INVALID, "too many pieces");
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(waves == 1 ? 256 : 64 * waves), 0, s, a);
    PKV_LAUNCH_CHECK();
    return PKV_OK;
  };
  auto by_rows = [&](auto type, auto dim) -> int {
    typedef decltype(type) T;
    constexpr int D = decltype(dim)::value;
    auto few = [&](auto waves) -> int {
      constexpr int N = decltype(waves)::value;
      return b.few_rows == 4   ? go(attend_4bit_kernel<T, D, 1, 4, N>, b.items, b.n_few, N)
             : b.few_rows == 8 ? go(attend_4bit_kernel<T, D, 1, 2, N>, b.items, b.n_few, N)
                               : go(attend_4bit_kernel<T, D, 1, 1, N>, b.items, b.n_few, N);
    };
    if (b.n_few) {
      const int rc = b.few_waves == 1 ? few(std::integral_constant<int, 1>{})
                                      : few(std::integral_constant<int, 4>{});
      if (rc) return rc;
    }
    if (b.n_wide) {
      const int rc = go(attend_4bit_kernel<T, D, 2, 1, 4>,
                        b.items + (int64_t)b.n_few * kPieceInts, b.n_wide, 4);
      if (rc) return rc;
    }
    if (b.n_tall)
      return run_4bit_tall(a, D, b.dtype, b.items + ((int64_t)b.n_few + b.n_wide) * kPieceInts,
                           b.n_tall, s);
    return PKV_OK;
  };
  auto by_dim = [&](auto type) -> int {
    return b.head_dim == 64 ? by_rows(type, std::integral_constant<int, 64>{})
                            : by_rows(type, std::integral_constant<int, 128>{});
  };
  return b.dtype == PKV_DTYPE_F16 ? by_dim(_Float16{}) : by_dim(__bf16{});
}

}  // extern "C"
