// The streaming decode kernel's body (decode.hip describes it): one workgroup
// of up to four waves runs a bin of a decode plan, a KV head a wave. shared.hip
// runs it beside tiles of shared pages in one launch.
#pragma once

#include "decode_piece.h"

namespace pkv {

#ifdef PKV_TIMELINE_KERNEL
// Instrumented build only (-DPKV_TIMELINE): every wave records, in 100 MHz
// s_memrealtime ticks, {start, first page done, last page done, end,
// pages, items, merges, ticks spent merging} with plain vector stores, for
// wave (bin * head groups + group) * waves + wave below kTimelineWaves. Read back with
// pkv_timeline_read.
constexpr int kTimelineWaves = 16384;
__device__ unsigned long long pkv_timeline[kTimelineWaves * 8];
#define PKV_TL(...) __VA_ARGS__
#else
#define PKV_TL(...)
#endif

// One wave's LDS tile: 16 K rows then 16 V rows of its head, each padded by
// 16 bytes so the K operand reads and the transposed V reads of a wave spread
// over the banks.
template <typename T, int D> struct Tile {
  static constexpr int RB = D * (int)sizeof(T);   // bytes of one head's row
  static constexpr int RS = RB + 16;
  static constexpr int BYTES = 2 * 16 * RS;
};

// A wave's item slots in LDS: C items of {Q rows of the G query heads of
// its KV head, the KV head's slice of the new K row, of the new V row}.
template <typename T, int D, int G> struct Stage {
  static constexpr int QB = G * D * (int)sizeof(T);
  static constexpr int RB = D * (int)sizeof(T);
  static constexpr int SLOT = QB + 2 * RB;
  static constexpr int C = 4096 / QB < 1 ? 1 : 4096 / QB > 8 ? 8 : 4096 / QB;
  static constexpr int QC = QB / 16;          // 16-byte chunks of the Q rows
  static constexpr int RC = RB / 16;          // of a new row slice
  static constexpr int CPI = SLOT / 16;       // per slot
  static constexpr int ROUNDS = (C * CPI + 63) / 64;
  static constexpr int BYTES = C * SLOT;
};

// A wave's two rings in LDS, for the stores it defers: KR new K/V row
// slices of its KV head (the fused append; RB2 bytes each) with their
// slots, and KO finished whole-sequence outputs (the rows of the G query
// heads of its KV head; OB bytes each) with their sequence ids. They share
// what a wave's share of 80 KiB leaves beside its tile and item slots (so
// two workgroups of four waves still fit a compute unit): the row ring up
// to half of it, the output ring the rest, each at most 16 entries. At
// head_dim 128 there is no row ring (KR = 0: the new rows are stored at
// once): its code would take the one-query-head kernel past 256 VGPRs, to
// one wave a SIMD.
template <typename T, int D, int G> struct Rings {
  static constexpr int OB = G * D * (int)sizeof(T);
  static constexpr int RB2 = 2 * D * (int)sizeof(T);
  static constexpr int FREE = 20480 - Tile<T, D>::BYTES - Stage<T, D, G>::BYTES - 2 * 64;
  static constexpr int KR0 = (FREE / 2 < FREE - OB ? FREE / 2 : FREE - OB) / RB2;
  static constexpr int KR = D > 64 ? 0 : KR0 < 1 ? 1 : KR0 > 16 ? 16 : KR0;
  static constexpr int KO0 = (FREE - KR * RB2) / OB;
  static constexpr int KO = KO0 < 1 ? 1 : KO0 > 16 ? 16 : KO0;
  static constexpr int ROWS = KR * RB2 + 64;     // row slices, then 16 slot ids
  static constexpr int BYTES = ROWS + KO * OB + 64;
};

// One workgroup per (bin, group of KV heads); wave w streams KV head
// hg * waves + w through the bin's pages, one piece (item) after another,
// without restarting the page pipeline at item boundaries. The bin's plan
// block at plan + bin * stride is {n_items, n_pages, 0, 0}, then n_pages page
// words (id | (live rows - 1) << 27 | bad << 31); its n_items items of
// kItemInts end the block, item i at plan + (bin + 1) * stride - (i + 1) *
// kItemInts. Header, first words and first items thus all sit at addresses
// known before any of them is read, so one round trip fetches them all and
// the first page and Q loads go out after it (the block is at least
// kHdrInts + kStageMax items long, so the first batch's item reads stay
// inside it).
//
// Cut sequences. A piece that is not its sequence's last publishes its
// partial (o, m, l) with sc1 stores and goes on streaming; its arrival is
// counted two pages later, when the wait for a page loaded after those
// stores has (vmcnt counts in order) also seen the stores complete, and the
// count it returns is checked at once. The last piece of a
// cut sequence runs at the end of its bin: it reads the arrival counter when
// it starts and, if every other piece has arrived by then, merges at its end
// without counting itself, its own partial taken from its registers (the
// same bits a store and a load would give, in the same place of the
// summation, so both paths produce the same output) and never stored;
// otherwise it publishes and counts its own arrival, and whichever piece
// arrives last merges.
//
// CHOSEN: the page words are not the plan's but each KV head's own, chosen on
// the device (selection.hip): head h's at `chosen` + h * head_words, where the
// plan has them.
template <typename T, int D, int G, bool CHOSEN = false>
__device__ __forceinline__ void decode_stream(
    unsigned char* smem, int bin, int group,
    const T* __restrict__ q, T* __restrict__ out, T* __restrict__ kpool, T* __restrict__ vpool,
    int64_t num_blocks, const int32_t* __restrict__ plan, int32_t stride, int32_t n_kv_heads,
    float scale_log2, const T* __restrict__ k_new, const T* __restrict__ v_new,
    const int32_t* __restrict__ slot_mapping, float* part_o, float* part_ml, uint32_t o_bytes,
    uint32_t ml_bytes, int32_t* counters, int32_t* status,
    const int32_t* __restrict__ chosen = nullptr, int64_t head_words = 0) {
  typedef typename Mma<T>::vec8 vec8;
  typedef typename Mma<T>::vec4 vec4;
  typedef PartLayout<D, G> PL;
  typedef Tile<T, D> TL;
  constexpr int PS = 16;
  constexpr int NCH = D / 32;          // QK MFMA k-chunks per head row
  constexpr int NDB = D / 16;          // PV MFMA dim blocks
  constexpr int RB = TL::RB;           // bytes of one head's row
  constexpr int CPR = RB / 16;         // 16-byte chunks per head row
  constexpr int RPI = 64 / CPR;        // rows per wave load instruction
  constexpr int NLD = PS / RPI;        // load instructions per page and tensor
  constexpr int RS = TL::RS;
  constexpr int NGR = PL::NGR;
  constexpr int OPS = 2 * NLD;         // vector memory instructions per page load
  static_assert(NLD * RPI == PS && CPR * RPI == 64, "a wave loads whole head rows");

  PKV_TL(const unsigned long long tl_start = __builtin_amdgcn_s_memrealtime();
         unsigned long long tl_first = 0, tl_merge = 0; int tl_merges = 0;)
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int hgw = heads_per_wg(n_kv_heads);          // KV heads of this workgroup (waves)
  const int h = group * hgw + wave;                  // this wave's KV head
  const int Hq = n_kv_heads * G;
  const uint32_t frow = (uint32_t)(n_kv_heads * RB);        // bytes per token row
  const int64_t row_elems = (int64_t)n_kv_heads * D;
  unsigned char* kl = smem + wave * TL::BYTES;       // this wave's tile: K rows
  unsigned char* vl = kl + PS * RS;                  // then V rows
  const int n = lane & 15;   // MFMA row/column within a 16-lane block
  const int g = lane >> 4;   // MFMA k-group

  const int32_t* bp = plan + (int64_t)bin * stride;
  const int32_t* words = bp + kHdrInts;
  if constexpr (CHOSEN)
    words = chosen + __builtin_amdgcn_readfirstlane(h) * head_words + (int64_t)bin * stride +
            kHdrInts;
  const int32_t* items_end = bp + stride;   // item i: items_end - (i + 1) * kItemInts
  typedef Stage<T, D, G> SG;
  static_assert(SG::C <= kStageMax, "the first batch's items lie inside the block");
  // read together with the header: the first batch's flags, the first item and
  // the first two page words
  int fl0[SG::C];
#pragma unroll
  for (int j = 0; j < SG::C; ++j) fl0[j] = items_end[-(j + 1) * kItemInts + 7];
  struct Item { int seq, np, tok0, kv, slot, nparts, slot0, flags; };
  auto item_at = [&](int i) __attribute__((always_inline)) -> Item {
    const int32_t* it = items_end - (int64_t)(i + 1) * kItemInts;
    return Item{it[0], it[1], it[2], it[3], it[4], it[5], it[6], it[7]};
  };
  Item cur = item_at(0);
  // the next item's fields, read one item ahead (the slot below a bin's last
  // item still lies inside its plan block: header and page words precede it)
  Item nxt = item_at(1);
  int wcur = words[0];
  int wnext = words[1];
  const int n_items = bp[0], n_pages = bp[1];
  // (keeps every one of these reads ahead of the branch below, so they go
  // out together instead of after it)
#pragma unroll
  for (int j = 0; j < SG::C; ++j) asm volatile("" ::"s"(fl0[j]));
  asm volatile("" ::"s"(cur.seq), "s"(cur.np), "s"(cur.tok0), "s"(cur.kv), "s"(cur.slot),
               "s"(cur.nparts), "s"(cur.slot0), "s"(cur.flags), "s"(wcur), "s"(wnext), "s"(q),
               "s"(k_new), "s"(v_new));
  if (n_items <= 0) return;

  // This lane's chunk of a page: row k * RPI + lane / CPR, bytes
  // (lane % CPR) * 16 of the head's slice -- CPR lanes cover a row, so every
  // load instruction reads whole cache lines.
  const int lrow0 = lane / CPR;
  const uint32_t lcol = (uint32_t)(lane % CPR) * 16;
  // Page p of the stream (p wave-uniform, word w = words[p]); past the
  // bin's last page every load is outside its range: no access, zeros.
  auto load_page = [&](int p, int w, vec8* kr, vec8* vr) __attribute__((always_inline)) {
    // (a plan's ids are checked on the host; chosen words are written on the device)
    const bool in = p < n_pages && (!CHOSEN || (w & ((1 << kPageIdBits) - 1)) < num_blocks);
    const int64_t page = in ? (w & ((1 << kPageIdBits) - 1)) : 0;
    const uint32_t live = in ? (((uint32_t)w >> kPageIdBits) & 15u) + 1u : 0u;
    const __amdgpu_buffer_rsrc_t rk = ws_rsrc(kpool + page * PS * row_elems, live * frow);
    const __amdgpu_buffer_rsrc_t rv = ws_rsrc(vpool + page * PS * row_elems, live * frow);
#pragma unroll
    for (int k = 0; k < NLD; ++k) {
      const uint32_t off = (uint32_t)(k * RPI + lrow0) * frow + (uint32_t)(h * RB) + lcol;
      kr[k] = __builtin_bit_cast(vec8, __builtin_amdgcn_raw_buffer_load_b128(rk, off, 0, kNt));
      vr[k] = __builtin_bit_cast(vec8, __builtin_amdgcn_raw_buffer_load_b128(rv, off, 0, kNt));
    }
  };
  // ---- items: fields from the plan (scalar loads); Q and the new row of
  // SG::C items at a time staged in this wave's LDS slots, loaded in one
  // batch (the first batch before the first pages, so waiting for it never
  // waits for a page).
  const bool fuse = k_new != nullptr;
  unsigned char* stg = smem + hgw * TL::BYTES + wave * SG::BYTES;
  // Loads of the slots of items i0 .. i0 + C - 1: lane chunk c = 64 r + lane
  // is 16 bytes w of item i's slot (Q rows of the KV head's G query heads,
  // then the KV head's slice of the new K row and of the new V row).
  // flags of items i0 .. i0 + C - 1 (the last item repeated past the end)
  auto stage_fields = [&](int i0, int* fl) __attribute__((always_inline)) {
    const int ns = min(SG::C, n_items - i0);
#pragma unroll
    for (int j = 0; j < SG::C; ++j)
      fl[j] = (items_end - (int64_t)(i0 + min(j, ns - 1) + 1) * kItemInts)[7];
  };
  auto stage_load = [&](int i0, const int* fl, u32x4* d) __attribute__((always_inline)) {
    const int ns = min(SG::C, n_items - i0);
#pragma unroll
    for (int r = 0; r < SG::ROUNDS; ++r) {
      const int c = r * 64 + lane;
      const int i = c / SG::CPI, w = c - i * SG::CPI;
      // item i's flags by masks (a select chain here becomes a lookup
      // table in scratch memory)
      int fi = 0;
#pragma unroll
      for (int j = 0; j < SG::C; ++j) fi |= fl[j] & -(int)(i == j);
      const int64_t ri = fi >> kRowShift;
      const unsigned char* src = nullptr;
      if (i < ns) {
        if (w < SG::QC)
          src = reinterpret_cast<const unsigned char*>(q + (ri * Hq + h * G) * D) + w * 16;
        else if (fuse && (fi & kItemLast))
          src = reinterpret_cast<const unsigned char*>(
                    (w < SG::QC + SG::RC ? k_new : v_new) + ri * row_elems + h * D) +
                (w < SG::QC + SG::RC ? w - SG::QC : w - SG::QC - SG::RC) * 16;
      }
      // each read once per item: streaming hint
      d[r] = src ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src))
                 : u32x4{0u, 0u, 0u, 0u};
    }
  };
  auto stage_store = [&](const u32x4* d) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < SG::ROUNDS; ++r) {
      const int c = r * 64 + lane;
      if (c < SG::C * SG::CPI) *reinterpret_cast<u32x4*>(stg + c * 16) = d[r];
    }
    wave_lds_sync();
  };
  u32x4 sgd[SG::ROUNDS];
  stage_load(0, fl0, sgd);
  // One page in flight: its registers and its word; the next page's word is
  // read a step ahead.
  vec8 kr[NLD], vr[NLD];
  load_page(0, wcur, kr, vr);
  stage_store(sgd);

  vec8 qb[NCH], kx{}, vx{};
  int new_slot = 0;
  // Item i (slot i % C staged) becomes current: Q^T as the QK B operand
  // (column n = query head h*G + n, zero beyond G) and this lane's 16 bytes
  // of the new row.
  auto take_item = [&](int i) __attribute__((always_inline)) {
    const unsigned char* sl = stg + (i % SG::C) * SG::SLOT;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const vec8 t = *reinterpret_cast<const vec8*>(
          sl + ((n < G ? n : 0) * D + c * 32 + g * 8) * (int)sizeof(T));
      qb[c] = (n < G) ? t : vec8{};
    }
    kx = *reinterpret_cast<const vec8*>(sl + SG::QB + lcol);
    vx = *reinterpret_cast<const vec8*>(sl + SG::QB + RB + lcol);
    new_slot = (fuse && (cur.flags & kItemLast)) ? slot_mapping[cur.flags >> kRowShift] : 0;
  };
  take_item(0);
  int it_idx = 0;
  int it_start = 0, it_end = cur.np;   // the current item's pages in the stream

  f32x4 o[NDB];
  float m_run = -INFINITY, l_run = 0.f;  // per head column n (replicated over g)
#pragma unroll
  for (int b = 0; b < NDB; ++b) o[b] = f32x4{0.f, 0.f, 0.f, 0.f};

  const __amdgpu_buffer_rsrc_t ro = ws_rsrc(part_o, o_bytes);
  const __amdgpu_buffer_rsrc_t rm = ws_rsrc(part_ml, ml_bytes);

  // Lane 4 g + i's value of v, in every lane of group g (heads 4 g + i < G;
  // other groups, whose rows are padding, get 1)
  auto from_lane = [&](float v, int i) __attribute__((always_inline)) {
    float x = 1.f;
#pragma unroll
    for (int gg = 0; 4 * gg < G; ++gg) {
      x = g == gg ? lane_value(v, 4 * gg + i) : x;
    }
    return x;
  };

  // Deferred stores. A whole sequence's output is normalised at the item's
  // end into the next entry of this wave's LDS output ring (lane (dim column
  // n, group g) holds heads 4g..4g+3 of dims 16b + n), and the fused
  // append's new row slices go to the row ring instead of the pool. A full
  // ring is stored in 16-byte pieces at the start of the next step, before
  // that step's page loads, and whatever the rings hold at the end of the
  // stream: a bin of many short sequences then writes in a few bursts
  // instead of a round of stores among the page reads at every item
  // (capacity phase A, 16 sequences a bin: 67.5 against 75.5 us a launch).
  // No other wave of the launch reads a new row's slot (the fusion's
  // precondition), and the kernel patches its own loaded copy at once, so
  // the deferral changes no result. Stores issued after a page's loads
  // would make the single wait at the top of the loop, which serves every
  // path, also wait for them; issued before them, they complete within the
  // wait for the page.
  typedef Rings<T, D, G> RG;
  unsigned char* rrow = smem + hgw * (TL::BYTES + SG::BYTES) + wave * RG::BYTES;
  int32_t* rrow_slot = reinterpret_cast<int32_t*>(rrow + RG::KR * RG::RB2);
  unsigned char* ring = rrow + RG::ROWS;
  int32_t* ring_seq = reinterpret_cast<int32_t*>(ring + RG::KO * RG::OB);
  int n_out = 0;    // outputs the output ring holds
  int n_rows = 0;   // row slices the row ring holds
  bool rows_full = false;
  // The row ring's first `cnt` entries to the pools: 16-byte piece c is
  // piece c % NCR of entry c / NCR (K slice, then V slice). Both rings are
  // written with the streaming hint: nothing in this launch reads them back.
  auto write_rows = [&](int cnt) __attribute__((always_inline)) {
    constexpr int NCR = RG::RB2 / 16;
    constexpr int HALF = NCR / 2;
#pragma unroll 1
    for (int c0 = 0; c0 < cnt * NCR; c0 += 64) {
      const int c = c0 + lane;
      if (c < cnt * NCR) {
        const int e = c / NCR, part = c - e * NCR;
        unsigned char* d = reinterpret_cast<unsigned char*>(
            (part < HALF ? kpool : vpool) + (int64_t)rrow_slot[e] * row_elems);
        __builtin_nontemporal_store(*reinterpret_cast<const u32x4*>(rrow + c * 16),
                                    reinterpret_cast<u32x4*>(d + h * RB + (part % HALF) * 16));
      }
    }
  };
  auto finish_out = [&]() __attribute__((always_inline)) {
    unsigned char* ol = ring + n_out * RG::OB;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * g + i;
      const float li = from_lane(l_run, i);  // lane r holds head r's sum
      if (r < G) {
        const float inv = 1.f / li;   // one division per row, not per element
#pragma unroll
        for (int b = 0; b < NDB; ++b)
          *reinterpret_cast<T*>(ol + (r * D + 16 * b + n) * (int)sizeof(T)) = (T)(o[b][i] * inv);
      }
    }
  };
  // The ring's first `cnt` rows to out: 16-byte piece c is piece c % NCK of
  // row c / NCK. (A rolled loop: unrolled, its loads stay live and cost
  // 30 VGPRs.)
  auto write_out = [&](int cnt) __attribute__((always_inline)) {
    constexpr int NCK = RG::OB / 16;
#pragma unroll 1
    for (int c0 = 0; c0 < cnt * NCK; c0 += 64) {
      const int c = c0 + lane;
      if (c < cnt * NCK) {
        const int row = c / NCK;
        T* dst = out + ((int64_t)ring_seq[row] * Hq + h * G) * D;
        __builtin_nontemporal_store(
            *reinterpret_cast<const u32x4*>(ring + c * 16),
            reinterpret_cast<u32x4*>(reinterpret_cast<unsigned char*>(dst) + (c - row * NCK) * 16));
      }
    }
  };
  bool ring_full = false;

  // The current item's last page: write the new row (fused append) and patch
  // the loaded copy when slot_mapping agrees with the page table.
  auto append_row = [&](int w, vec8* kq, vec8* vq) __attribute__((always_inline)) {
    const int tl = (cur.kv - 1) % PS;  // newest token's row within its page
    const int64_t page = w & ((1 << kPageIdBits) - 1);
    const bool in_range = new_slot >= 0 && (int64_t)new_slot < num_blocks * PS;
    if (!in_range) {
      if (lane == 0) flag(status, PKV_STATUS_BAD_SLOT);
      return;
    }
    const bool patch = (int64_t)new_slot == page * PS + tl;
    if constexpr (RG::KR > 0) {   // into the row ring's next entry
      unsigned char* e = rrow + n_rows * RG::RB2;
      if (lane == 0) rrow_slot[n_rows] = new_slot;
      rows_full = ++n_rows == RG::KR;
#pragma unroll
      for (int k = 0; k < NLD; ++k) {
        if (k * RPI + lrow0 == tl) {
          *reinterpret_cast<vec8*>(e + lcol) = kx;
          *reinterpret_cast<vec8*>(e + RB + lcol) = vx;
          if (patch) {
            kq[k] = kx;
            vq[k] = vx;
          }
        }
      }
    } else {                      // into the pools at once
      unsigned char* kd = reinterpret_cast<unsigned char*>(kpool + new_slot * row_elems);
      unsigned char* vd = reinterpret_cast<unsigned char*>(vpool + new_slot * row_elems);
#pragma unroll
      for (int k = 0; k < NLD; ++k) {
        if (k * RPI + lrow0 == tl) {
          *reinterpret_cast<vec8*>(kd + h * RB + lcol) = kx;
          *reinterpret_cast<vec8*>(vd + h * RB + lcol) = vx;
          if (patch) {
            kq[k] = kx;
            vq[k] = vx;
          }
        }
      }
    }
  };

  // Merge (seq, h) from the stored partials and reset its counter.
  auto merge = [&](int sq, int orow, int nparts, int slot0, bool own) __attribute__((always_inline)) {
    PKV_TL(const unsigned long long tm = __builtin_amdgcn_s_memrealtime(); ++tl_merges;)
    merge_head<T, D, G>(out, reinterpret_cast<float*>(kl), orow, h, n_kv_heads, nparts, slot0,
                        ro, rm, own, o, m_run, l_run);
    if (lane == 0)
      __hip_atomic_store(counters + (int64_t)sq * n_kv_heads + h, 0, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    PKV_TL(tl_merge += __builtin_amdgcn_s_memrealtime() - tm;)
  };
  // Count an arrival whose partial has completed; the returned count.
  auto arrive = [&](int sq) __attribute__((always_inline)) -> int {
    int old = 0;
    if (lane == 0)
      old = __hip_atomic_fetch_add(counters + (int64_t)sq * n_kv_heads + h, 1, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
    return old;
  };
  // A deferred arrival: pa_state 1 once a partial is stored; it is counted
  // at page pa_at.
  int pa_state = 0, pa_at = 0, pa_seq = 0, pa_row = 0, pa_nparts = 0, pa_slot0 = 0, pa_old = 0;
  // check a counted arrival: the last one merges
  auto finish_arrival = [&]() __attribute__((always_inline)) {
    if (__builtin_amdgcn_readfirstlane(pa_old) == pa_nparts - 1)
      merge(pa_seq, pa_row, pa_nparts, pa_slot0, false);
    pa_state = 0;
  };
  auto flush_arrival = [&]() __attribute__((always_inline)) {  // count a pending arrival now
    if (pa_state == 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      pa_old = arrive(pa_seq);
      finish_arrival();
    }
  };
  int b_count = 0;   // the arrival counter as the last piece of a cut sequence found it

  // Item end: the output (whole sequence), or the partial of a cut sequence.
  auto end_item = [&](int p) __attribute__((always_inline)) {
    if (cur.slot < 0) {
      finish_out();
      if (lane == 0) ring_seq[n_out] = cur.flags >> kRowShift;
      ring_full = ++n_out == RG::KO;
    } else {
      flush_arrival();   // at most one deferred arrival at a time
      const bool last = cur.flags & kItemLast;
      if (last && __builtin_amdgcn_readfirstlane(b_count) == cur.nparts - 1) {
        // the sequence's last piece, and every other piece had arrived when
        // it started: it merges, its own partial straight from registers,
        // and publishes nothing
        merge(cur.seq, cur.flags >> kRowShift, cur.nparts, cur.slot0, true);
      } else {
        const uint32_t head_off =
            (uint32_t)(((int64_t)cur.slot * n_kv_heads + h) * PL::FLOATS * 4);
        if (g < NGR) {
#pragma unroll
          for (int b = 0; b < NDB; ++b)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o[b]), ro,
                                                   head_off + ((g * NDB + b) * 16 + n) * 16, 0,
                                                   kSc1);
        }
        if (lane < G)
          __builtin_amdgcn_raw_buffer_store_b64(
              __builtin_bit_cast(u32x2, f32x2{m_run, l_run}), rm,
              (uint32_t)(((int64_t)cur.slot * Hq + h * G + lane) * 8), 0, kSc1);
        asm volatile("" ::: "memory");  // the stores stay before the loads that follow
        pa_seq = cur.seq;
        pa_row = cur.flags >> kRowShift;
        pa_nparts = cur.nparts;
        pa_slot0 = cur.slot0;
        if (!last && p + 2 < n_pages) {
          // count it once a page loaded after the stores has arrived
          pa_state = 1;
          pa_at = p + 2;
        } else {
          // the last piece with others still out, or the stream ends: count
          // it now; whichever piece arrives last merges
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          pa_old = arrive(cur.seq);
          finish_arrival();
        }
      }
    }
    ++it_idx;
    if (it_idx < n_items) {
      if (it_idx % SG::C == 0) {   // the next batch of slots
        int fl[SG::C];
        stage_fields(it_idx, fl);
        stage_load(it_idx, fl, sgd);
        stage_store(sgd);
      }
      cur = nxt;
      nxt = item_at(it_idx + 1);
      take_item(it_idx);
      it_start = it_end;
      it_end += cur.np;
      m_run = -INFINITY;
      l_run = 0.f;
#pragma unroll
      for (int b = 0; b < NDB; ++b) o[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };

  auto compute = [&](int p) __attribute__((always_inline)) {
    const int tp = cur.tok0 + (p - it_start) * PS;  // first token of the page
    // S^T: lane (n, g) gets the scores of tokens 4g..4g+3 for head n.
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const unsigned char* kp = kl + n * RS + g * 16;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      acc = Mma<T>::qk(*reinterpret_cast<const vec8*>(kp + c * 64), qb[c], acc);
    float sc[4];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sc[i] = tp + 4 * g + i < cur.kv ? acc[i] * scale_log2 : -INFINITY;
      mx = fmaxf(mx, sc[i]);
    }
    mx = max_x32(max_x16(mx));
    // Lazy rescale: the reference max moves only when some head's max
    // grows by more than 2^8, so p <= 256 and o / l is unchanged.
    if (__builtin_amdgcn_ballot_w64(mx > m_run + 8.f)) {
      const float m_new = fmaxf(m_run, mx);  // finite: every page has a live token
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
      m_run = m_new;
      // lane (n, g) holds output rows 4g+i, whose factor lives in lane 4g+i
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = from_lane(alpha, i);
#pragma unroll
        for (int b = 0; b < NDB; ++b) o[b][i] *= a;
      }
    }
    vec4 pr;
    float ls = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = __builtin_amdgcn_exp2f(sc[i] - m_run);
      ls += e;
      pr[i] = (T)e;
    }
    ls = sum_x32(sum_x16(ls));
    l_run += ls;
    const unsigned char* vp = vl + (4 * g + (n >> 2)) * RS + 4 * (n & 3) * (int)sizeof(T);
#pragma unroll
    for (int b = 0; b < NDB; ++b) {
      const i16x4 raw = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_i16x4*)(vp + 16 * b * sizeof(T)));
      o[b] = Mma<T>::pv(pr, __builtin_bit_cast(vec4, raw), o[b]);
    }
  };

  // Step p: stage page p into the wave's tile (patched with the new row at
  // a sequence's last page), send the loads of page p + 1 into the same
  // registers, then compute page p. Every step issues exactly one page's
  // loads (past the bin's last page: no access), so on every path through
  // the loop the wait for page p counts only page p's loads.
  for (int p = 0; p < n_pages; ++p) {
    if (fuse && (cur.flags & kItemLast) && p == it_end - 1) append_row(wcur, kr, vr);
    if (wcur < 0 && lane == 0) flag(status, PKV_STATUS_BAD_PAGE);
#pragma unroll
    for (int k = 0; k < NLD; ++k) {
      const uint32_t loff = (uint32_t)(k * RPI + lrow0) * RS + lcol;
      *reinterpret_cast<vec8*>(kl + loff) = kr[k];
      *reinterpret_cast<vec8*>(vl + loff) = vr[k];
    }
    wave_lds_sync();
    if (RG::KR > 0 && rows_full) {   // full rings, before this step's loads
      write_rows(RG::KR);
      rows_full = false;
      n_rows = 0;
    }
    if (ring_full) {
      write_out(RG::KO);
      ring_full = false;
      n_out = 0;
    }
    if (p == it_start && (cur.flags & kItemLast) && cur.slot >= 0 && lane == 0)
      b_count = __hip_atomic_load(counters + (int64_t)cur.seq * n_kv_heads + h,
                                  __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wcur = wnext;
    wnext = words[p + 2];   // inside the plan block: its words are followed by items
    load_page(p + 1, wcur, kr, vr);
    compute(p);
    PKV_TL(if (p == 0) tl_first = __builtin_amdgcn_s_memrealtime();)
    // (after compute: a merge below uses the wave's tile as scratch)
    if (pa_state != 0 && p == pa_at) {
      // Page p's loads were issued after the partial's stores and have
      // arrived (vmcnt counts in order); only page p + 1's loads may still
      // be outstanding, so this wait leaves the stores complete.
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OPS) : "memory");
      pa_old = arrive(pa_seq);
      finish_arrival();
    }
    if (p == it_end - 1) end_item(p);
    wave_lds_sync();  // this page's tile reads are done before the next copy
  }
  PKV_TL(const unsigned long long tl_last = __builtin_amdgcn_s_memrealtime();)
  if (n_rows + n_out > 0) wave_lds_sync();   // the last entries and their ids
  if (RG::KR > 0 && n_rows > 0) write_rows(n_rows);
  if (n_out > 0) write_out(n_out);
  flush_arrival();
#ifdef PKV_TIMELINE_KERNEL
  {
    const int wid = (blockIdx.y * gridDim.x + blockIdx.x) * hgw + wave;
    const unsigned long long tl_end = __builtin_amdgcn_s_memrealtime();
    if (lane < 8 && wid < kTimelineWaves) {
      const unsigned long long rec[8] = {tl_start, tl_first, tl_last, tl_end,
                                         (unsigned long long)n_pages, (unsigned long long)n_items,
                                         (unsigned long long)tl_merges, tl_merge};
      unsigned long long v = rec[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) v = lane == i ? rec[i] : v;
      pkv_timeline[(int64_t)wid * 8 + lane] = v;
    }
  }
#endif
}

template <typename T, int D, int G>
static size_t decode_lds_bytes(int hgw) {
  return (size_t)hgw * (Tile<T, D>::BYTES + Stage<T, D, G>::BYTES + Rings<T, D, G>::BYTES);
}

}  // namespace pkv
