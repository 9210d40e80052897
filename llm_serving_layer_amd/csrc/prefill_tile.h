// Chunked-prefill attention over a paged prefix on gfx950 matrix cores.
//
// One workgroup (4 waves) owns one KV head h and one tile of a sequence's
// query rows: 128 rows = BQ query tokens x G query heads (BQ = 128 / G), so
// every K/V tile it loads serves all G query heads of the KV head. Each wave
// owns 32 rows. Query row r of the tile is token r / G (of the tile) and
// query head h*G + r % G; it sits at absolute position kv_len - q_len +
// token (bottom-right causal alignment, as the reference's
// triu(diagonal = kv_len - q_len + 1) mask) and sees keys 0..position.
//
// The KV axis is walked 32 tokens (two pages) at a time. A tile of K and of
// V (those rows x head_dim of head h) goes straight from memory into one of
// four LDS buffers (a ring; direct-to-LDS buffer loads two tiles ahead, each
// wave one page of one tensor, rows unpadded with their 16-byte chunks
// swizzled) and is read by every wave. All products are 32x32x16 MFMAs, so every LDS byte read feeds 32
// query rows:
//  * S^T = K Q^T: K rows from LDS as the A operand, Q^T held in registers
//    as the B operand. Lane (row n, group g) gets 16 scores of its query row
//    n: keys 8 i + 4 g + 0..3, i = 0..3;
//  * online softmax per query row, lane-local; the two half-waves holding a
//    row meet (v_permlane32_swap) only for a row max and for the final sum;
//  * O^T = V^T P^T: V^T from transposing LDS reads as the A operand, the
//    lane's own 8 probabilities of a 16-key block as the B operand (the
//    contraction index runs over keys 4 g + 0..3, 8 + 4 g + 0..3 of the
//    block). Every O^T accumulator of a lane belongs to its own query row,
//    so rescaling needs no cross-lane traffic.
// The running reference moves lazily: probabilities are taken against it,
// and only when some lane's sum of a tile's probabilities passes 2^12 is
// the row max taken and the accumulators rescaled, so probabilities stay at
// most 2^12 and o / l is unchanged. Tiles wholly below the causal diagonal
// skip the mask. Each wave's share of a tile lies within one page, so page
// ids are scalar reads and pages are buffer ranges: rows past kv_len read
// zeros without a memory access.
// Numerics as serving/backends/paged_torch.py:443-485: scores, softmax and
// accumulation in fp32; probabilities rounded to the pool dtype before PV.
// The scale must be positive (the row max is taken before scaling); other
// scales run the generic kernel.
#pragma once

#include "mfma.h"

namespace pkv {

constexpr int kPrefillRows = 128;   // query rows per workgroup (tokens x heads)
constexpr int kPrefillThreads = 256; // 4 waves x 32 rows

typedef float f32x16 __attribute__((ext_vector_type(16)));
template <typename T> struct Mma32;
template <> struct Mma32<_Float16> {
  __device__ static f32x16 mma(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mma32<__bf16> {
  __device__ static f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// LDS of one workgroup: a ring of four K/V tile buffers, rows unpadded with
// 16-byte chunks XOR-swizzled by row.
template <typename T, int D> struct PrefillLds {
  static constexpr int TT = 32;                        // KV tokens per tile
  static constexpr int RB = D * (int)sizeof(T);        // bytes of one head's row
  static constexpr int TILE = TT * RB;                 // one K (or V) tile
  static constexpr int BYTES = 4 * 2 * TILE;
  static constexpr int LPT = TILE / 2 / 1024;          // wave loads of a page of one tensor
};

// Lane 4 k + i of v[e] becomes lane 4 k + e of v[i]: a 4 x 4 transpose in every
// quad of lanes (a swap of pairs a lane apart, then of pairs two apart).
__device__ __forceinline__ f32x4 quad_transpose(f32x4 v) {
  const int lane = threadIdx.x;
  const bool a = lane & 1, b = lane & 2;
  f32x4 t;
#pragma unroll
  for (int e = 0; e < 4; e += 2) {   // quad_perm [1,0,3,2]
    const float x = dpp<0xB1>(a ? v[e] : v[e + 1]);
    t[e] = a ? x : v[e];
    t[e + 1] = a ? v[e + 1] : x;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {      // quad_perm [2,3,0,1]
    const float x = dpp<0x4E>(b ? t[e] : t[e + 2]);
    v[e] = b ? x : t[e];
    v[e + 2] = b ? t[e + 2] : x;
  }
  return v;
}

// A tile over pages that several one-token sequences share (shared.hip): its
// rows are those sequences' queries, all of which see every key, and its
// result is a partial (o, m, l) per sequence, in the decode kernels' layout.
struct SharedTile {
  const int32_t* items;      // {first page in kv_indices, pages, first member, members, split}
  const int32_t* members;    // {row of q, partial slot of split 0}
  float* part_o;
  float* part_ml;
};
constexpr int kSharedItem = 8, kSharedMember = 2;   // ints of each

// The swizzle of a shared tile's rows (16-byte chunk c of row r at chunk
// position c ^ wide_xr(r)): LDS hands 256 bytes a cycle to 16 lanes of a 16-byte
// read, or 32 of an 8-byte one. 16 rows read at one chunk (K) and four rows,
// from a multiple of four on, at four chunks, from a multiple of four on (V),
// then meet 16 different positions of the 256 bytes; a row of 128 bytes is half
// of them. (By the eight-row swizzle of the other kernels half of the LDS
// cycles were bank conflicts.)
template <int RB> __device__ __forceinline__ int wide_xr(int row) {
  return RB == 128 ? ((row >> 1) & 1) << 2 | ((row >> 2) & 3) : (row & 3) << 2 | ((row >> 2) & 3);
}

// A shared tile's ring: four slots of a K and a V tile, 64 KiB (two workgroups a
// compute unit), K loaded three tiles ahead and V as far ahead of its use. Such a
// tile has at most one more workgroup beside it, so its own loads have to cover
// the memory's latency, where a prefill tile's neighbours do.
// At head_dim 64 a tile has 64 keys: a step's fixed cost (scalar instructions, a
// barrier, the wait for the first LDS reads) is paid half as often, and two score
// products run side by side.
template <typename T, int D> struct SharedRing {
  static constexpr int TT = D == 64 ? 64 : 32;              // keys of a tile
  static constexpr int TILE = TT * D * (int)sizeof(T);      // one K (or V) tile
  static constexpr int N = 4;
  static constexpr int BYTES = N * 2 * TILE;
};

template <typename T, int D, int G, bool SHARED = false>
__device__ __forceinline__ void prefill_tile(
    unsigned char* smem, int block,
    const T* __restrict__ q, T* __restrict__ out, const T* __restrict__ kpool,
    const T* __restrict__ vpool, int64_t num_blocks, const int32_t* __restrict__ cu_q,
    const int32_t* __restrict__ kv_indptr, const int32_t* __restrict__ kv_indices,
    const int32_t* __restrict__ kv_lens, const int32_t* __restrict__ plan,
    int32_t n_kv_heads, float scale_log2, int32_t* status, const SharedTile& sh = SharedTile{}) {
  typedef typename Mma<T>::vec8 vec8;
  typedef typename Mma<T>::vec4 vec4;
  typedef PrefillLds<T, D> L;
  constexpr int TT = SHARED ? SharedRing<T, D>::TT : L::TT;
  constexpr int TILE = SHARED ? SharedRing<T, D>::TILE : L::TILE;
  constexpr int PS = 16;
  constexpr int NH = TT / 32;            // 32-key halves per tile
  constexpr int NC = D / 16;             // QK k-chunks of 16 dims
  constexpr int NDH = D / 32;            // PV blocks of 32 dims
  constexpr int RB = L::RB;
  constexpr int CPR = RB / 16;           // 16-byte chunks per row
  constexpr int LPT = L::LPT;
  static_assert(64 % CPR == 0 && PS % (64 / CPR) == 0, "a wave load stays in one page");
  unsigned char* const buf0 = smem + 0 * 2 * TILE;
  unsigned char* const buf1 = smem + 1 * 2 * TILE;
  unsigned char* const buf2 = smem + 2 * 2 * TILE;
  unsigned char* const buf3 = smem + 3 * 2 * TILE;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int n = lane & 31, g = lane >> 5;
  const int item = block / n_kv_heads;
  const int h = block - item * n_kv_heads;
  int qs = 0, qn, q0 = 0, kv_len, pbase, base_pos;
  const int32_t* members = nullptr;
  int split = 0;
  if constexpr (SHARED) {
    const int32_t* it = sh.items + (int64_t)item * kSharedItem;
    pbase = it[0];
    kv_len = it[1] * PS;
    members = sh.members + (int64_t)it[2] * kSharedMember;
    qn = it[3];
    split = it[4];
    base_pos = kv_len - 1;      // every row sees every key
  } else {
    const int seq = plan[4 * item];
    qs = plan[4 * item + 1];
    qn = plan[4 * item + 2];
    q0 = cu_q[seq];
    const int q_len = cu_q[seq + 1] - q0;
    kv_len = kv_lens[seq];
    pbase = kv_indptr[seq];
    base_pos = kv_len - q_len + qs;
  }
  const int Hq = n_kv_heads * G;
  const int64_t row = (int64_t)n_kv_heads * D;
  const int kv_end = SHARED ? kv_len : base_pos + qn;
  const int ntiles = (kv_end + TT - 1) / TT;

  // This lane's query row (column n of every 32x32 tile) and Q^T as the B
  // operand of S^T = K Q^T: lane (n, g) holds Q[row][16c + 8g .. + 7].
  const int r = wave * 32 + n;
  const int tok = r / G;
  const bool valid = tok < qn;
  const int qpos = valid && !SHARED ? base_pos + tok : kv_len - 1;
  vec8 qb[NC];
  {
    int token = q0 + qs + (valid ? tok : 0);
    if constexpr (SHARED) token = members[(valid ? tok : 0) * kSharedMember];
    const T* qr = q + ((int64_t)token * Hq + h * G + r % G) * D + g * 8;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const vec8 t = *reinterpret_cast<const vec8*>(qr + c * 16);
      qb[c] = valid ? t : vec8{};
    }
  }

  // A wave loads one page of one tensor of a tile, 16 rows of the KV head: one
  // buffer range to set up instead of one per page and tensor (about 45 scalar
  // instructions a step instead of 130; a 777-token prompt, head_dim 128, 8
  // layers with their appends: 205 -> 195 us, with the ring no longer zeroed
  // at the start; no change where four waves share a SIMD). The page id is
  // read with a scalar load a tile ahead. (Scalar loads, so the vector-memory count holds
  // tile loads only: a plain vector load may complete before a direct-to-LDS
  // load issued earlier, so the count cannot prove a tile landed if the two
  // mix.)
  const int npages = (kv_len + PS - 1) / PS;
  const uint32_t rowbytes = (uint32_t)(row * sizeof(T));
  const uint32_t pagebytes = PS * rowbytes;
  // ids at or past this are out of range (kv_indices entries are int32)
  const uint32_t nb32 = num_blocks > 0x7fffffffLL ? 0x80000000u : (uint32_t)num_blocks;
  // (a tile of four pages: a wave loads one page of both tensors)
  constexpr bool BOTH = TT == 4 * PS;
  static_assert(BOTH || TT == 2 * PS, "a tile is two pages or four");
  const int wpage = BOTH ? wave : wave & 1;
  const T* const wpool = BOTH || wave < 2 ? kpool : vpool;
  const uint32_t wdst = (BOTH || wave < 2 ? 0 : TILE) + wpage * PS * RB;
  constexpr int RPI = 64 / CPR;                  // rows of a wave load
  uint32_t voff[LPT];
#pragma unroll
  for (int k = 0; k < LPT; ++k) {
    const int rr = k * RPI + lane / CPR;
    const int lc = SHARED ? (lane % CPR) ^ wide_xr<RB>(rr)
                          : ((lane % CPR) ^ xr(rr)) & 7 | ((lane % CPR) & ~7);
    voff[k] = (uint32_t)rr * rowbytes + (uint32_t)(h * RB + lc * 16);
  }
  auto load_id = [&](int t) {   // this wave's page id for tile t
    return __builtin_amdgcn_readfirstlane(kv_indices[pbase + min(TT / PS * t + wpage, npages - 1)]);
  };
  // Rows past kv_len, pages past the last and out-of-range pages are outside
  // the buffer range: zeros land in LDS without a memory access.
  auto load_tile = [&](int t, int raw, const unsigned char* dst) {
    const int pg = TT / PS * t + wpage;
    const bool bad = (uint32_t)raw >= nb32;   // (negative ids too)
    if (bad && pg < npages && lane == 0) flag(status, PKV_STATUS_BAD_PAGE);
    const int live_rows = bad ? 0 : min(PS, kv_len - pg * PS);   // <= 0 past the end
    const uint32_t pid = bad ? 0u : (uint32_t)raw;
    load_to_lds<LPT>(
        raw_rsrc(reinterpret_cast<const char*>(wpool) + (uint64_t)pid * pagebytes,
                 live_rows > 0 ? (uint32_t)live_rows * rowbytes : 0u),
        voff, lds_address(dst) + wdst);
    if constexpr (BOTH)
      load_to_lds<LPT>(
          raw_rsrc(reinterpret_cast<const char*>(vpool) + (uint64_t)pid * pagebytes,
                   live_rows > 0 ? (uint32_t)live_rows * rowbytes : 0u),
          voff, lds_address(dst) + wdst + TILE);
  };

  // O^T accumulators: o[dh][rr] = O[row][32 dh + 8 (rr / 4) + 4 g + rr % 4].
  f32x16 o[NDH];
#pragma unroll
  for (int dh = 0; dh < NDH; ++dh) o[dh] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  // the transposing V reads: lane i of each 16-lane block points at key
  // (i / 4) of a 4-key group and dims 4 (i % 4) .. + 3 of its 16-dim block
  const int vrow = lane & 15;
  const int vcol = (lane & 16) + 4 * (vrow & 3);

  // element e of row `row` of a tile
  auto in_tile = [&](int row, int e) __attribute__((always_inline)) {
    return SHARED ? row * RB + ((e >> 3) ^ wide_xr<RB>(row)) * 16 + (e & 7) * 2 : swz<RB>(row, e);
  };
  // P^T of the previous tile (the B operand of its PV), kept for the next step.
  vec8 pb[NH * 2];
#pragma unroll
  for (int i = 0; i < NH * 2; ++i) pb[i] = vec8{};
  // O^T += V^T P^T for a tile: V^T as the A operand, lane (dim, g) holding
  // V[key][dim] for keys 16 kb + 4 g + 0..3 and 16 kb + 8 + 4 g + 0..3.
  auto read_v = [&](const unsigned char* vl, vec8* va) {
#pragma unroll
    for (int kb = 0; kb < NH * 2; ++kb) {
      const int key = 16 * kb + 4 * g + (vrow >> 2);
#pragma unroll
      for (int dh = 0; dh < NDH; ++dh) {
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_i16x4*)(vl + in_tile(key, vcol + 32 * dh)));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_i16x4*)(vl + in_tile(key + 8, vcol + 32 * dh)));
        va[kb * NDH + dh] = __builtin_bit_cast(
            vec8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    }
  };
  auto pv_mma = [&](const vec8* va) {
#pragma unroll
    for (int kb = 0; kb < NH * 2; ++kb) {
#pragma unroll
      for (int dh = 0; dh < NDH; ++dh) o[dh] = Mma32<T>::mma(va[kb * NDH + dh], pb[kb], o[dh]);
    }
  };
  auto pv = [&](const unsigned char* vl) {
    vec8 va[NH * 2 * NDH];
    read_v(vl, va);
    pv_mma(va);
  };

  // Tile t: S^T = K Q^T, then its softmax beside the previous tile's PV
  // (independent of it), which leaves tile t's probabilities in pb.
  auto compute = [&](int t, const unsigned char* kl, const unsigned char* vprev) {
    const int t0 = t * TT;
    const bool full = t0 + TT - 1 <= base_pos;
    // the previous tile's V operands, read while QK runs
    vec8 va[NH * 2 * NDH];
    // S^T = K Q^T: s[hf][rr] = score of key t0 + 32 hf + 8 (rr / 4) + 4 g + rr % 4.
    f32x16 s[NH];
    read_v(vprev, va);
#pragma unroll
    for (int hf = 0; hf < NH; ++hf) {
      s[hf] = f32x16{};
      const int kr = hf * 32 + n;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        s[hf] = Mma32<T>::mma(*reinterpret_cast<const vec8*>(kl + in_tile(kr, 16 * c + 8 * g)),
                              qb[c], s[hf]);
    }
    // Keys past the row's position are masked only on tiles that reach them.
    if (!full) {
#pragma unroll
      for (int hf = 0; hf < NH; ++hf) {
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) {
          const int key = t0 + 32 * hf + 8 * (rr >> 2) + 4 * g + (rr & 3);
          if (key > qpos) s[hf][rr] = -INFINITY;
        }
      }
    }
    // The previous tile's PV (zero probabilities before the first tile), its
    // matrix instructions interleaved with the softmax's vector ones below.
    pv_mma(va);
    // Probabilities against the running reference m_run: 16-key block
    // (hf, qq) of P^T uses the lane's scores rr = 8 qq .. 8 qq + 7 in that
    // order.
    float ls = 0.f;
    auto probs = [&]() {
      ls = 0.f;
#pragma unroll
      for (int hf = 0; hf < NH; ++hf) {
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[hf][rr], scale_log2, -m_run));
          ls += e;
          pb[2 * hf + (rr >> 3)][rr & 7] = (T)e;
        }
      }
    };
    probs();
    // (pinned here: otherwise the compiler moves them behind the max test)
#pragma unroll
    for (int i = 0; i < NH * 2; ++i) {
      u32x4 w = __builtin_bit_cast(u32x4, pb[i]);
      asm volatile("" : "+v"(w));
      pb[i] = __builtin_bit_cast(vec8, w);
    }
    asm volatile("" : "+v"(ls));
#pragma unroll
    for (int i = 0; i < NH * 2 * NDH; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // one MFMA
      __builtin_amdgcn_sched_group_barrier(0x002, 12, 0);  // then vector work
    }
    // Lazy rescale: the reference only moves when some lane's sum of its
    // probabilities passes 2^12, which bounds every one of them by 2^12
    // (within the pool dtype's range; NaN or inf counts as past it, as on the
    // first tile, whose reference is -inf); the result o / l does not depend
    // on which reference is used. Only then is the row max taken: it is at
    // least 8 above the reference (a sum past 2^12 over 16 keys has a term
    // past 2^8), so the reference grows, o (with the previous tile's PV
    // added) and l are rescaled and the probabilities taken again.
    if (__builtin_amdgcn_ballot_w64(!(ls <= 4096.f))) {
      // raw-score row max (scale_log2 > 0, so scaling commutes with max)
      float mx = -INFINITY;
#pragma unroll
      for (int hf = 0; hf < NH; ++hf) {
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) mx = fmaxf(mx, s[hf][rr]);
      }
      mx = max_x32(mx) * scale_log2;
      const float m_new = fmaxf(m_run, mx);   // finite: key 0 is visible to every row
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int dh = 0; dh < NDH; ++dh) o[dh] *= alpha;
      probs();
    }
    // l_run: this lane's half of its row's keys; the halves meet at the end
    l_run += ls;
  };

  unsigned char* last = buf0;   // the buffer of the last tile computed
  if constexpr (SHARED) {
    // Three tiles are at work in a step, none waiting for another: tile t's
    // scores and tile t - 2's PV on the matrix cores, tile t - 1's softmax on
    // the vector unit. K of tile t is in slot t % N of the ring, V in the V half
    // of the same slot; a step loads K of tile t + AHEAD and V of tile t - 2 +
    // AHEAD, into the slots that step t - 1 was the last to read.
    // One wave a SIMD is bound by its instructions, scalar ones too, so the
    // steps are unrolled over the slots (constant LDS offsets) and a step's
    // loads need few: page ids from a vector register, 64 tiles' at a time. At
    // head_dim 128 a step has 141 instructions and takes 1250 cycles, 512 of them
    // the matrix cores' part; with 267 instructions it took 1600 (128 sequences
    // over 1024 pages, 8 KV heads of 128: the tiles alone 55 -> 45 us, beside the
    // own pages and with the merge 83 -> 71).
    constexpr int N = SharedRing<T, D>::N, AHEAD = N - 1, TP = TT / PS;
    static_assert(N == 4, "the steps below are unrolled over four slots");
    auto k_slot = [&](int i) { return smem + (i & (N - 1)) * 2 * TILE; };
    auto v_slot = [&](int i) { return smem + (i & (N - 1)) * 2 * TILE + TILE; };
    const uint32_t lds0 = lds_address(smem) + wdst;   // (wdst: this wave's page; V's half)
    uint32_t vnext[LPT];                              // voff without load k's offset
#pragma unroll
    for (int k = 0; k < LPT; ++k) vnext[k] = voff[k] - 1024 * k;
    uint32_t worst = 0;                               // of the page ids, unsigned
    auto load_page = [&](const T* pool, uint32_t id, int left, uint32_t at) {
      worst = max(worst, id);
      load_page_to_lds<LPT>(raw_rsrc(reinterpret_cast<const char*>(pool) + (uint64_t)id * pagebytes,
                                     id < nb32 && left > 0 ? pagebytes : 0u),
                            vnext, at);
    };
    // A wave that loads V alone is two tiles behind. Lane l: this wave's page of
    // tile 64 c + l - behind.
    const int behind = !BOTH && wave >= 2 ? 2 : 0;
    const int first_page = wpage - behind * TP;
    int page_ids;
    auto read_ids = [&](int j) {
      page_ids = kv_indices[pbase + max(0, min(TP * (j + lane) + first_page, npages - 1))];
    };
    uint32_t id1 = 0, id2 = 0;                        // (BOTH) of tiles j - 1, j - 2
    // K of tile j into slot j % N, V of tile j - 2 into its slot; none before tile 0
    auto load_step = [&](int j, auto to, bool v_too) {
      constexpr int S = decltype(to)::value;
      const uint32_t id = __builtin_amdgcn_readlane(page_ids, j & 63);
      const int left = npages - first_page - TP * j;  // pages from this wave's on
      constexpr uint32_t k_at = S * 2 * TILE, v_at = ((S + N - 2) % N) * 2 * TILE;
      if constexpr (BOTH) {
        load_page(kpool, id, left, lds0 + k_at);
        load_page(vpool, id2, v_too ? left + 2 * TP : 0, lds0 + v_at + TILE);
        id2 = id1;
        id1 = id;
      } else {
        load_page(wpool, id, behind && !v_too ? 0 : left, lds0 + (behind ? v_at : k_at));
      }
    };
    template_for<0, AHEAD>([&](auto j) {
      if constexpr (decltype(j)::value == 0) read_ids(0);
      load_step(j, j, decltype(j)::value >= 2);
    });
#pragma unroll
    for (int c = 0; c < NC; ++c) {   // Q arrives here (see below)
      u32x4 w = __builtin_bit_cast(u32x4, qb[c]);
      asm volatile("" : "+v"(w));
      qb[c] = __builtin_bit_cast(vec8, w);
    }
    auto arrive = [&]() {            // tiles t (K) and t - 2 (V) are in their slots
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((AHEAD - 1) * LPT * (BOTH ? 2 : 1)) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    typedef vec8 Keys[NH * NC];
    typedef f32x16 Scores[NH];
    typedef vec8 Probs[NH * 2];
    auto read_k = [&](const unsigned char* kl, Keys& ka) {
#pragma unroll
      for (int hf = 0; hf < NH; ++hf)
#pragma unroll
        for (int c = 0; c < NC; ++c)
          ka[hf * NC + c] =
              *reinterpret_cast<const vec8*>(kl + in_tile(hf * 32 + n, 16 * c + 8 * g));
      asm volatile("" ::: "memory");
    };
    auto qk = [&](const Keys& ka, Scores& s) {
#pragma unroll
      for (int hf = 0; hf < NH; ++hf) s[hf] = f32x16{};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int hf = 0; hf < NH; ++hf) s[hf] = Mma32<T>::mma(ka[hf * NC + c], qb[c], s[hf]);
    };
    auto pv_of = [&](const vec8* va, const Probs& p) {
#pragma unroll
      for (int kb = 0; kb < NH * 2; ++kb)
#pragma unroll
        for (int dh = 0; dh < NDH; ++dh) o[dh] = Mma32<T>::mma(va[kb * NDH + dh], p[kb], o[dh]);
    };
    // (Probabilities are rounded to the pool's type: the matrix product takes no
    // other. As in attend; 256 sequences in fp16 differ from 64 bits by 3.0e-4 of
    // the outputs' norm, 2.1e-4 where probabilities keep 32: there all of it is the
    // output's own rounding.)
    auto softmax = [&](const Scores& s, Probs& p, float& ls) {
      ls = 0.f;
#pragma unroll
      for (int hf = 0; hf < NH; ++hf)
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[hf][rr], scale_log2, -m_run));
          ls += e;
          p[2 * hf + (rr >> 3)][rr & 7] = (T)e;
        }
    };
    // the lazy rescale of compute() above, with tile t - 2's PV in o
    auto settle = [&](const Scores& s, Probs& p, float ls) {
      if (__builtin_amdgcn_ballot_w64(!(ls <= 4096.f))) {
        float mx = -INFINITY;
#pragma unroll
        for (int hf = 0; hf < NH; ++hf)
#pragma unroll
          for (int rr = 0; rr < 16; ++rr) mx = fmaxf(mx, s[hf][rr]);
        mx = max_x32(mx) * scale_log2;
        const float m_new = fmaxf(m_run, mx);
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
        m_run = m_new;
#pragma unroll
        for (int dh = 0; dh < NDH; ++dh) o[dh] *= alpha;
        softmax(s, p, ls);
      }
      l_run += ls;
    };
    auto pin = [&](Probs& p, float& ls) {   // (not behind the test)
#pragma unroll
      for (int i = 0; i < NH * 2; ++i) {
        u32x4 w = __builtin_bit_cast(u32x4, p[i]);
        asm volatile("" : "+v"(w));
        p[i] = __builtin_bit_cast(vec8, w);
      }
      asm volatile("" : "+v"(ls));
    };
    constexpr int FIRST = 20, EACH = 3;
    // Step t, t % N == S: scores of tile t into s1, the softmax of tile t - 1's
    // (s0) into p1, PV of tile t - 2 (p0).
    auto step = [&](int t, auto slot, const Scores& s0, Scores& s1, const Probs& p0, Probs& p1) {
      constexpr int S = decltype(slot)::value;
      arrive();
      Keys ka;
      vec8 va[NH * 2 * NDH];
      read_k(k_slot(S), ka);
      read_v(v_slot(S + N - 2), va);
      asm volatile("" ::: "memory");
      load_step(t + AHEAD, std::integral_constant<int, (S + AHEAD) % N>{}, true);
      qk(ka, s1);
      pv_of(va, p0);
      float ls;
      softmax(s0, p1, ls);
      pin(p1, ls);
      // vector work while the LDS reads are on their way, then beside each MFMA
      __builtin_amdgcn_sched_group_barrier(0x002, FIRST * NH, 0);
#pragma unroll
      for (int i = 0; i < NH * NC + NH * 2 * NDH; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, EACH * NH, 0);
      }
      settle(s0, p1, ls);
    };
    // The last tile's softmax, with its missing keys, and the last two PVs.
    auto drain = [&](Scores& s0, const Probs& p0, Probs& p1) {
      arrive();
      vec8 va[NH * 2 * NDH];
      read_v(v_slot(ntiles - 2 + N), va);
      if (ntiles * TT > kv_len) {
#pragma unroll
        for (int hf = 0; hf < NH; ++hf)
#pragma unroll
          for (int rr = 0; rr < 16; ++rr)
            if ((ntiles - 1) * TT + 32 * hf + 8 * (rr >> 2) + 4 * g + (rr & 3) >= kv_len)
              s0[hf][rr] = -INFINITY;
      }
      pv_of(va, p0);
      float ls;
      softmax(s0, p1, ls);
      settle(s0, p1, ls);
      // (all loads, those of the tiles past the end too, before the workgroup ends)
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      read_v(v_slot(ntiles - 1), va);
      pv_of(va, p1);
    };
    Scores sa, sb;
    Probs pa, pz;
#pragma unroll
    for (int i = 0; i < NH * 2; ++i) pa[i] = vec8{};
    {
      arrive();
      load_step(AHEAD, std::integral_constant<int, AHEAD>{}, true);
      Keys ka;
      read_k(k_slot(0), ka);
      qk(ka, sa);
    }
    auto swap = [&]() {   // an odd number of steps: back to sa and pa
#pragma unroll
      for (int hf = 0; hf < NH; ++hf) sa[hf] = sb[hf];
#pragma unroll
      for (int i = 0; i < NH * 2; ++i) pa[i] = pz[i];
    };
    for (int t = 1;; t += 4) {
      if (t >= ntiles) break;
      if (((t + AHEAD) & 63) == 0) read_ids(t + AHEAD);
      step(t, std::integral_constant<int, 1>{}, sa, sb, pa, pz);
      if (t + 1 >= ntiles) { swap(); break; }
      step(t + 1, std::integral_constant<int, 2>{}, sb, sa, pz, pa);
      if (t + 2 >= ntiles) break;
      step(t + 2, std::integral_constant<int, 3>{}, sa, sb, pa, pz);
      if (t + 3 >= ntiles) { swap(); break; }
      step(t + 3, std::integral_constant<int, 0>{}, sb, sa, pz, pa);
    }
    drain(sa, pa, pz);
    if (worst >= nb32 && lane == 0) flag(status, PKV_STATUS_BAD_PAGE);
  } else {
    // The ring: tile t in buffer t % 4. Each step waits for its tile's loads
    // (this wave's, then every wave's at the barrier, which also ends every
    // wave's reads of the buffer the step then refills: the one of tile t - 2,
    // whose PV ran in the previous step), loads the pages of tile t + 2,
    // computes tile t beside the PV of tile t - 1, and loads the page ids of
    // tile t + 3.
    // The first step's PV meets zero probabilities in buf3, which no tile has
    // filled yet: zeros there (visible to every wave at the step's barrier).
    for (int i = tid; i < TILE / 16; i += kPrefillThreads)
      reinterpret_cast<u32x4*>(buf3 + TILE)[i] = u32x4{0u, 0u, 0u, 0u};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    int id0 = load_id(0), id1 = load_id(1), id2 = load_id(2), id3;   // of tile j in id(j % 4)
    load_tile(0, id0, buf0);
    load_tile(1, id1, buf1);
    // Q arrives here: waited for inside the loop, where the compiler cannot see
    // the tile loads, it would drain them in every step
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      u32x4 w = __builtin_bit_cast(u32x4, qb[c]);
      asm volatile("" : "+v"(w));
      qb[c] = __builtin_bit_cast(vec8, w);
    }
    auto step = [&](int t, unsigned char* cur, unsigned char* prev, unsigned char* nxt2,
                    int& id_t2, int& id_t3) {
      // Every tile load but the latest step's has landed; after the barrier,
      // every wave's have. (A fenced barrier would wait for all of them.)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LPT) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      load_tile(t + 2, id_t2, nxt2);
      compute(t, cur, prev + TILE);
      // (after the tile's LDS reads: a scalar load in flight would make every
      // wait for them a wait for it too)
      id_t3 = load_id(t + 3);
    };
    for (int t = 0;; t += 4) {
      step(t, buf0, buf3, buf2, id2, id3);
      last = buf0;
      if (t + 1 >= ntiles) break;
      step(t + 1, buf1, buf0, buf3, id3, id0);
      last = buf1;
      if (t + 2 >= ntiles) break;
      step(t + 2, buf2, buf1, buf0, id0, id1);
      last = buf2;
      if (t + 3 >= ntiles) break;
      step(t + 3, buf3, buf2, buf1, id1, id2);
      last = buf3;
      if (t + 4 >= ntiles) break;
    }
  }
  if constexpr (!SHARED) {
    pv(last + TILE);   // the last tile's PV
    // the loads of the tiles past the end land in LDS before the workgroup ends
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  l_run = sum_x32(l_run);
  if constexpr (SHARED) {
    // The partial of the row's sequence and head: groups of four heads, a
    // float4 over them per dim. Four heads are four lanes here, so a quad of
    // lanes transposes its four dims (j & 3) into one 16-byte store each: a
    // quad then writes 64 bytes in a row. (Below four heads the groups are
    // padded, and each lane stores its own.)
    constexpr int NDB = D / 16, FLOATS = (G + 3) / 4 * NDB * 64;
    const int hd = r % G;
    const int32_t* mb = members + (valid ? tok : 0) * kSharedMember;
    const int64_t slot = mb[1] + split;
    float* po = sh.part_o + (slot * n_kv_heads + h) * FLOATS + (hd / 4) * NDB * 64;
#pragma unroll
    for (int dh = 0; dh < NDH; ++dh) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 v{o[dh][4 * j], o[dh][4 * j + 1], o[dh][4 * j + 2], o[dh][4 * j + 3]};
        const int d0 = 32 * dh + 8 * j + 4 * g;
        if constexpr (G >= 4) {
          v = quad_transpose(v);   // lane hd & 3: dim d0 + (hd & 3) of the group's heads
          if (valid) *reinterpret_cast<f32x4*>(po + (d0 + (hd & 3)) * 4) = v;
        } else if (valid) {
#pragma unroll
          for (int e = 0; e < 4; ++e) po[(d0 + e) * 4 + hd] = v[e];
        }
      }
    }
    if (valid && g == 0)
      *reinterpret_cast<f32x2*>(sh.part_ml + (slot * Hq + h * G + hd) * 2) = f32x2{m_run, l_run};
    return;
  }
  if (valid) {
    const float inv = 1.f / l_run;
    T* orow = out + ((int64_t)(q0 + qs + tok) * Hq + h * G + r % G) * D + 4 * g;
#pragma unroll
    for (int dh = 0; dh < NDH; ++dh) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        vec4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(o[dh][4 * j + e] * inv);
        *reinterpret_cast<vec4*>(orow + 32 * dh + 8 * j) = v;
      }
    }
  }
}

}  // namespace pkv
