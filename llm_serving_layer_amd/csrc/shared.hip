// Decode attention for sequences that begin with the same pages: each shared
// run of pages is read once for all of them instead of once each.
//
// A softmax over a sequence's keys splits over any partition of them: part j
// leaves m_j = max s, l_j = sum e^(s - m_j), o_j = sum e^(s - m_j) v, and the
// whole is sum_j w_j o_j / sum_j w_j l_j, w_j = e^(m_j - max m). Page lists that
// begin alike form a tree; each of its inner runs is one part of every sequence
// below it, and its own pages are the sequence's last part (its last page
// always is its own, so every sequence has one).
//  * A run is a prefill tile's work (prefill_tile.h): the queries of the
//    sequences that share it are its 128 rows, so a tile of K and V loaded once
//    serves 128 / G sequences on the matrix cores. Long runs are split over
//    workgroups. Each leaves its parts in the decode kernels' partial slots.
//  * The own pages are pieces of a decode plan, as pieces of cut sequences
//    whose other parts are the shared ones.
//  * Both run in one launch, side by side: the tiles are bound by the matrix
//    cores, the own pages by memory, and a compute unit holds a workgroup of
//    each. Tiles count no arrivals, so nobody in that launch knows when a
//    sequence's parts are complete; a last small launch merges them.
#include <algorithm>
#include <exception>
#include <numeric>
#include <vector>

#include "decode_stream.h"
#include "prefill_tile.h"

namespace pkv {

template <typename T> struct SharedArgs {
  const T* q; T* out; T* kp; T* vp;
  int64_t nb; const int32_t* indices; int32_t Hkv; float sl2; SharedTile sh;
  const int32_t* plan; int32_t stride; const T* kn; const T* vn; const int32_t* slots;
  DecodeWorkspace w; int32_t* status;
  int32_t tiles, pieces, turn;   // workgroups of each kind, and in a row of one kind
};

// The launch's workgroup `block` as one of the tiles (>= 0) or of the pieces
// (~ of its number): the kinds take turns, `turn` at a time, as long as both
// have that many, then the rest of the tiles and of the pieces follow.
__device__ __forceinline__ int shared_role(int block, int tiles, int pieces, int turn) {
  const int rounds = min(tiles, pieces) / turn, both = rounds * 2 * turn;
  if (block < both) {
    const int round = block / (2 * turn), at = block - round * 2 * turn;
    return at < turn ? round * turn + at : ~(round * turn + at - turn);
  }
  const int at = block - both + rounds * turn;
  return at < tiles ? at : ~(at - tiles + rounds * turn);
}

// Tiles beside the bins of the streaming decode kernel (four KV heads a bin's
// workgroup, a wave each: bins of fewer run in a launch of their own).
template <typename T, int D, int G>
__global__ __launch_bounds__(256, 2) void shared_stream_kernel(SharedArgs<T> a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int role = shared_role(blockIdx.x, a.tiles, a.pieces, a.turn);
  if (role >= 0) {
    prefill_tile<T, D, G, true>(smem, role, a.q, nullptr, a.kp, a.vp, a.nb, nullptr, nullptr,
                                a.indices, nullptr, nullptr, a.Hkv, a.sl2, a.status, a.sh);
  } else {
    const int groups = a.Hkv / heads_per_wg(a.Hkv), bin = ~role / groups;
    decode_stream<T, D, G>(smem, bin, ~role - bin * groups, a.q, a.out, a.kp, a.vp, a.nb, a.plan,
                           a.stride, a.Hkv, a.sl2, a.kn, a.vn, a.slots, a.w.part_o, a.w.part_ml,
                           a.w.o_bytes, a.w.ml_bytes, a.w.counters, a.status);
  }
}

// Tiles beside the small-batch decode kernel's workgroups, one a piece and KV head.
template <typename T, int D, int G>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void shared_piece_kernel(SharedArgs<T> a) {
  constexpr int A = PieceLds<T, D, G>::BYTES, B = SharedRing<T, D>::BYTES;
  __shared__ __align__(16) unsigned char smem[A > B ? A : B];
  const int role = shared_role(blockIdx.x, a.tiles, a.pieces, a.turn);
  if (role >= 0) {
    prefill_tile<T, D, G, true>(smem, role, a.q, nullptr, a.kp, a.vp, a.nb, nullptr, nullptr,
                                a.indices, nullptr, nullptr, a.Hkv, a.sl2, a.status, a.sh);
  } else {
    const int bin = ~role / a.Hkv;
    decode_piece<T, D, G>(smem, ~role - bin * a.Hkv, bin, a.q, a.out, a.kp, a.vp, a.nb, a.plan,
                          a.stride, a.Hkv, a.sl2, a.kn, a.vn, a.slots, a.w.part_o, a.w.part_ml,
                          a.w.o_bytes, a.w.ml_bytes, a.w.counters, a.status);
  }
}

// The merge of every sequence with shared parts: a wave a KV head; it clears the
// arrivals that the sequence's own pieces counted.
template <typename T, int D, int G>
__global__ __launch_bounds__(64) void shared_merge_kernel(T* out, const int32_t* list,
                                                          int32_t n_kv_heads, DecodeWorkspace w) {
  constexpr int NGR = PartLayout<D, G>::NGR;
  __shared__ __align__(16) float wts[64 * 4 * NGR];
  const int i = blockIdx.x / n_kv_heads, h = blockIdx.x - i * n_kv_heads;
  const int32_t* it = list + (int64_t)i * 4;   // {sequence, parts, first slot, 0}
  const int seq = it[0], parts = it[1], slot0 = it[2];
  f32x4 none[D / 16];
#pragma unroll
  for (int b = 0; b < D / 16; ++b) none[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  merge_head<T, D, G>(out, wts, seq, h, n_kv_heads, parts, slot0, ws_rsrc(w.part_o, w.o_bytes),
                      ws_rsrc(w.part_ml, w.ml_bytes), false, none, 0.f, 0.f);
  if (threadIdx.x == 0) w.counters[(int64_t)seq * n_kv_heads + h] = 0;
}

struct SharedLaunch {
  const void* q; void* out; void* kp; void* vp; int64_t nb; const int32_t* indices; int32_t Hkv;
  float sl2; SharedTile sh; int32_t n_tiles; const int32_t* list; int32_t n_list;
  const int32_t* plan; int32_t n_work, stride; const void* kn; const void* vn;
  const int32_t* slots; DecodeWorkspace w; int32_t* status; int32_t dtype;
};

// The decode launch of a plan (decode.hip).
void run_decode(int32_t dtype, int32_t D, int32_t G, const void* q, void* out, void* kp, void* vp,
                int64_t nb, const int32_t* plan, int32_t n_work, int32_t stride, int32_t Hkv,
                float sl2, const void* kn, const void* vn, const int32_t* slots,
                const DecodeWorkspace& w, int32_t* status, hipStream_t s);

template <typename T, int D, int G>
static void launch_shared(const SharedLaunch& l, hipStream_t s) {
  const int groups = l.Hkv / heads_per_wg(l.Hkv);
  const bool few = few_pieces(l.n_work, l.stride, l.Hkv, D);
  SharedArgs<T> a{(const T*)l.q, (T*)l.out, (T*)l.kp, (T*)l.vp, l.nb, l.indices, l.Hkv, l.sl2, l.sh,
                  l.plan, l.stride, (const T*)l.kn, (const T*)l.vn, l.slots, l.w,
                  l.status, l.n_tiles * l.Hkv, few ? l.n_work / groups * l.Hkv : l.n_work,
                  std::max(1, compute_units())};
  // A bin's workgroup has a wave a KV head, four at most. With fewer than four
  // it would leave the launch's other waves idle beside it, so it gets a launch
  // of its own behind the tiles'.
  const bool apart = !few && heads_per_wg(l.Hkv) < kMaxWaves;
  if (apart) a.pieces = 0;
  const dim3 grid((unsigned)(a.tiles + a.pieces));
  if (few) {
    hipLaunchKernelGGL((shared_piece_kernel<T, D, G>), grid, dim3(256), 0, s, a);
  } else {
    const size_t lds = std::max<size_t>(decode_lds_bytes<T, D, G>(heads_per_wg(l.Hkv)),
                                        SharedRing<T, D>::BYTES);
    hipLaunchKernelGGL((shared_stream_kernel<T, D, G>), grid, dim3(256), lds, s, a);
  }
  if (apart)
    run_decode(l.dtype, D, G, l.q, l.out, l.kp, l.vp, l.nb, l.plan, l.n_work, l.stride, l.Hkv,
               l.sl2, l.kn, l.vn, l.slots, l.w, l.status, s);
  hipLaunchKernelGGL((shared_merge_kernel<T, D, G>), dim3((unsigned)(l.n_list * l.Hkv)), dim3(64),
                     0, s, a.out, l.list, l.Hkv, l.w);
}

typedef void (*SharedFn)(const SharedLaunch&, hipStream_t);

template <typename T, int D>
static SharedFn shared_g(int G) {
  switch (G) {
    case 1: return launch_shared<T, D, 1>;
    case 2: return launch_shared<T, D, 2>;
    case 4: return launch_shared<T, D, 4>;
    case 8: return launch_shared<T, D, 8>;
    case 16: return launch_shared<T, D, 16>;
    default: return nullptr;
  }
}

static SharedFn shared_fn(int32_t dtype, int32_t D, int32_t G) {
  if (dtype == PKV_DTYPE_F16)
    return D == 64 ? shared_g<_Float16, 64>(G) : D == 128 ? shared_g<_Float16, 128>(G) : nullptr;
  if (dtype == PKV_DTYPE_BF16)
    return D == 64 ? shared_g<__bf16, 64>(G) : D == 128 ? shared_g<__bf16, 128>(G) : nullptr;
  return nullptr;
}

int check_geometry(int32_t Hq, int32_t Hkv, int32_t D, int32_t ps, int32_t dtype);
int check_seq_pages(int32_t i, int32_t np, int32_t kv, int32_t last, int32_t ps);
int split_workspace(void* workspace, int64_t workspace_bytes, int32_t n_seqs, int32_t n_slots,
                    int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, DecodeWorkspace* w);

namespace {

// A run of pages [first, last) of the members' lists, which they share.
struct Run {
  int32_t first, last;
  std::vector<int32_t> members;
};

// The runs of the tree of page lists, of at least min_pages pages and two
// members, that save more than they cost: all but one member's reads of the run
// against a part more of each member; `own` marks per kv_indices entry the pages that stay a sequence's own.
struct Tree {
  const int32_t* indptr;
  const int32_t* indices;
  int32_t min_pages;
  int64_t page_bytes, part_bytes;   // of a KV head
  std::vector<Run> runs;
  std::vector<char> own;

  int64_t saved(int64_t members, int64_t pages) const {
    return (members - 1) * pages * page_bytes - members * part_bytes;
  }

  int32_t room(int32_t i) const { return indptr[i + 1] - indptr[i] - 1; }   // the last page is own
  int32_t page(int32_t i, int32_t p) const { return indices[indptr[i] + p]; }

  void grow(int32_t n_seqs) {
    own.assign(indptr[n_seqs], 1);
    std::vector<Run> open(1);   // runs whose members may share more pages behind them
    open[0].first = open[0].last = 0;
    open[0].members.resize(n_seqs);
    std::iota(open[0].members.begin(), open[0].members.end(), 0);
    while (!open.empty()) {
      const Run run = std::move(open.back());
      open.pop_back();
      const int32_t at = run.last;
      std::vector<int32_t> m;
      for (int32_t i : run.members)
        if (room(i) > at) m.push_back(i);
      std::stable_sort(m.begin(), m.end(),
                       [&](int32_t a, int32_t b) { return page(a, at) < page(b, at); });
      for (size_t a = 0, b; a < m.size(); a = b) {
        for (b = a + 1; b < m.size() && page(m[b], at) == page(m[a], at);) ++b;
        if (b - a < 2) continue;
        const int32_t* lead = indices + indptr[m[a]];
        int32_t end = room(m[a]);
        for (size_t j = a + 1; j < b; ++j) {
          const int32_t* mine = indices + indptr[m[j]];
          end = std::min(end, room(m[j]));
          end = (int32_t)(std::mismatch(lead + at, lead + end, mine + at).first - lead);
        }
        Run child{at, end, std::vector<int32_t>(m.begin() + a, m.begin() + b)};
        if (end - at >= min_pages && saved((int64_t)(b - a), end - at) >= 0) {
          for (int32_t i : child.members)
            std::fill(own.begin() + indptr[i] + at, own.begin() + indptr[i] + end, 0);
          runs.push_back(child);
        }
        open.push_back(std::move(child));
      }
    }
  }
};

}  // namespace
}  // namespace pkv

using namespace pkv;

extern "C" int pkv_plan_shared(const int32_t* kv_indptr, const int32_t* kv_indices,
                               const int32_t* kv_lens, const int32_t* kv_last_page_len,
                               int32_t n_seqs, int32_t page_size, int64_t num_blocks,
                               int32_t n_heads, int32_t n_kv_heads, int32_t part_pages,
                               int32_t max_workgroups, int32_t min_pages, int64_t page_bytes,
                               int64_t part_bytes, int64_t least_bytes, int32_t tile_target,
                               int32_t* plan, int64_t plan_capacity, int64_t* plan_needed,
                               int32_t* n_work_out, int32_t* n_slots_out,
                               int32_t* plan_stride_out, int32_t* tiles, int64_t tiles_capacity,
                               int64_t* tiles_needed, int32_t* n_tiles_out,
                               int32_t* n_merges_out) try {
  if (n_seqs <= 0 || page_size <= 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads)
    return fail(PKV_ERR_INVALID, "n_seqs, page_size and heads must be positive, n_heads a "
                "multiple of n_kv_heads");
  const int32_t G = n_heads / n_kv_heads;
  if (G > kPrefillRows || kPrefillRows % G || min_pages < 1 || tile_target < 1)
    return fail(PKV_ERR_INVALID, "%d query heads a KV head, min_pages=%d or tile_target=%d is "
                "not supported", G, min_pages, tile_target);
  if (kv_indptr[0] != 0) return fail(PKV_ERR_INVALID, "kv_indptr must start at 0");
  for (int32_t i = 0; i < n_seqs; ++i) {
    const int rc = check_seq_pages(i, kv_indptr[i + 1] - kv_indptr[i], kv_lens[i],
                                   kv_last_page_len[i], page_size);
    if (rc) return rc;
  }
  Tree tree{kv_indptr, kv_indices, min_pages, page_bytes, part_bytes, {}, {}};
  tree.grow(n_seqs);
  int64_t saved = 0;
  for (const Run& r : tree.runs)
    saved += n_kv_heads * tree.saved((int64_t)r.members.size(), r.last - r.first);
  if (plan_needed) *plan_needed = 0;
  if (tiles_needed) *tiles_needed = 0;
  if (tree.runs.empty() || saved < least_bytes) {
    *n_work_out = *n_slots_out = *plan_stride_out = *n_tiles_out = *n_merges_out = 0;
    return PKV_OK;
  }

  // The own pages as a batch of their own, planned by pkv_plan_decode. (Only
  // the number of a sequence's keys matters to a one-token query, not where
  // they stand, so its own pages count from 0.)
  std::vector<int32_t> ptr(n_seqs + 1, 0), ids, lens(n_seqs);
  ids.reserve(kv_indptr[n_seqs]);
  for (int32_t i = 0; i < n_seqs; ++i) {
    for (int32_t p = kv_indptr[i]; p < kv_indptr[i + 1]; ++p)
      if (tree.own[p]) ids.push_back(kv_indices[p]);
    ptr[i + 1] = (int32_t)ids.size();
    lens[i] = (ptr[i + 1] - ptr[i] - 1) * page_size + kv_last_page_len[i];
  }
  // Runs in splits of about `split` pages: from 8 on, so that no more than
  // tile_target workgroups share the work (or one each, where that is more), and
  // so that a tile takes about as long as the own pages beside it: 180 of those
  // (times KV heads) stream in the time a tile takes for one page (at 250 and 130:
  // 96 sequences, 256 shared pages, 4 KV heads of 128: 39.5 and 33.6 us; 128
  // sequences, 1024 shared pages, 8 KV heads of 128: 70.5 and 84.4). Shorter tiles
  // only leave more parts to merge (96 sequences, 7 runs of 32 and 49 pages,
  // head_dim 128: 36.0 us with 30 tiles, 31.5 with 9).
  const int32_t per_tile = kPrefillRows / G;
  int64_t steps = 0;   // pages times row tiles, over all runs
  int32_t longest = 0;
  for (const Run& r : tree.runs) {
    steps += (int64_t)(r.last - r.first) * ((r.members.size() + per_tile - 1) / per_tile);
    longest = std::max(longest, r.last - r.first);
  }
  const int64_t target = std::max<int64_t>(1, tile_target / n_kv_heads);
  int64_t split = std::max<int64_t>({8, (steps + target - 1) / target,
                                     (int64_t)ids.size() * n_kv_heads / 180});
  auto splits_of = [&](const Run& r) {   // (rounded, and at least one)
    const int32_t n = r.last - r.first;
    return (int32_t)std::max<int64_t>(1, (n + split / 2) / split);
  };
  // a run's split sizes: equal, an even number (a tile's step is two pages or four)
  auto size_of = [&](const Run& r) {
    const int32_t n = r.last - r.first, k = splits_of(r);
    return ((n + k - 1) / k + 1) / 2 * 2;
  };
  for (; split < longest; split += 2) {
    int64_t tiles_now = 0;
    for (const Run& r : tree.runs)
      tiles_now += (int64_t)splits_of(r) * ((r.members.size() + per_tile - 1) / per_tile);
    if (tiles_now <= target) break;
  }
  std::vector<int32_t> shared(n_seqs, 0);   // shared parts of each sequence
  int64_t n_tiles = 0, n_members = 0;
  for (const Run& r : tree.runs) {
    const int32_t size = size_of(r), splits = (r.last - r.first + size - 1) / size;
    n_tiles += splits * (int64_t)((r.members.size() + per_tile - 1) / per_tile);
    n_members += (int64_t)r.members.size();
    for (int32_t i : r.members) shared[i] += splits;
  }
  const int32_t n_merges = (int32_t)std::count_if(shared.begin(), shared.end(),
                                                  [](int32_t x) { return x > 0; });
  // Two workgroups a compute unit (2 tile_target) are resident, tiles among them:
  // with bins for all of those the last bins began when the first workgroups had
  // ended (256 sequences, 64 tiles, head_dim 64: 47.3 us with 512, 39.1 with 448).
  const bool beside = heads_per_wg(n_kv_heads) == kMaxWaves;   // (else a launch of their own)
  const int32_t bins_wgs = beside ? (int32_t)std::min<int64_t>(max_workgroups, std::max<int64_t>(
      tile_target, 2 * (int64_t)tile_target - n_tiles * n_kv_heads)) : max_workgroups;
  int32_t n_work = 0, own_slots = 0, stride = 0;
  int64_t need = 0;
  int rc = pkv_plan_decode(ptr.data(), ids.data(), lens.data(), kv_last_page_len, n_seqs, page_size,
                           num_blocks, n_kv_heads, part_pages, bins_wgs, plan, plan_capacity,
                           &need, &n_work, &own_slots, &stride);
  if (plan_needed) *plan_needed = need;
  if (rc) return rc;

  // items and merges of 8 and 4 ints, members of 2
  const int64_t want = n_tiles * kSharedItem + (int64_t)n_merges * 4 + n_members * kSharedMember;
  if (tiles_needed) *tiles_needed = want;
  if (want > tiles_capacity || n_tiles * n_kv_heads > 0x7fffffffLL)
    return fail(PKV_ERR_CAPACITY, "shared tiles need %lld entries, capacity %lld",
                (long long)want, (long long)tiles_capacity);

  // Partial slots: a sequence's shared parts, then its own pieces.
  std::vector<int32_t> pieces(n_seqs, 1), base(n_seqs + 1, 0);
  const int64_t bins = n_work / (n_kv_heads / heads_per_wg(n_kv_heads));
  auto each_item = [&](auto&& f) {
    for (int64_t b = 0; b < bins; ++b)
      for (int32_t j = 0; j < plan[b * stride]; ++j)
        f(plan + (b + 1) * stride - (int64_t)(j + 1) * kItemInts);
  };
  each_item([&](int32_t* it) { pieces[it[0]] = it[4] < 0 ? 1 : it[5]; });
  for (int32_t i = 0; i < n_seqs; ++i) {
    const int32_t parts = shared[i] + pieces[i];
    base[i + 1] = base[i] + (parts > 1 ? parts : 0);
  }
  each_item([&](int32_t* it) {
    const int32_t i = it[0], parts = shared[i] + pieces[i];
    if (parts < 2) return;
    const int32_t ord = it[4] < 0 ? 0 : it[4] - it[6];
    it[4] = base[i] + shared[i] + ord;
    it[5] = parts;
    it[6] = base[i];
  });

  // Merges; tiles and members, a run's members in order, 128 / G of them a tile.
  int32_t* item = tiles;
  int32_t* merge = tiles + n_tiles * kSharedItem;
  int32_t* member = merge + (int64_t)n_merges * 4;
  for (int32_t i = 0; i < n_seqs; ++i) {
    if (!shared[i]) continue;
    const int32_t vals[4] = {i, shared[i] + pieces[i], base[i], 0};
    merge = std::copy(vals, vals + 4, merge);
  }
  int32_t at = 0;
  std::vector<int32_t> next(base.begin(), base.end() - 1);   // each sequence's next shared slot
  for (const Run& r : tree.runs) {
    const int32_t size = size_of(r), splits = (r.last - r.first + size - 1) / size;
    const int32_t n = (int32_t)r.members.size();
    for (int32_t s = 0; s < splits; ++s) {
      const int32_t first = r.first + s * size, pages = std::min(size, r.last - first);
      for (int32_t m = 0; m < n; m += per_tile) {
        const int32_t vals[kSharedItem] = {kv_indptr[r.members[0]] + first, pages, at + m,
                                           std::min(per_tile, n - m), s, 0, 0, 0};
        item = std::copy(vals, vals + kSharedItem, item);
      }
    }
    for (int32_t i : r.members) {
      const int32_t vals[kSharedMember] = {i, next[i]};
      member = std::copy(vals, vals + kSharedMember, member);
      next[i] += splits;
    }
    at += n;
  }
  *n_work_out = n_work;
  *n_slots_out = base[n_seqs];
  *plan_stride_out = stride;
  *n_tiles_out = (int32_t)n_tiles;
  *n_merges_out = n_merges;
  return PKV_OK;
} catch (const std::exception& e) {   // (no memory for the plan: nothing leaves a C entry)
  return fail(PKV_ERR_CAPACITY, "pkv_plan_shared: %s", e.what());
}

extern "C" int pkv_attend_shared(const void* q, void* out, void* k_pool, void* v_pool,
                                 int64_t num_blocks, const int32_t* kv_indices, int32_t n_seqs,
                                 int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                 int32_t page_size, float scale, int32_t dtype,
                                 const int32_t* tiles, int32_t n_tiles, int32_t n_merges,
                                 const int32_t* plan, int32_t n_work, int32_t n_slots, int32_t plan_stride,
                                 const void* k_new, const void* v_new,
                                 const int32_t* slot_mapping, void* workspace,
                                 int64_t workspace_bytes, int32_t* status_word, void* stream) {
  int rc = check_geometry(n_heads, n_kv_heads, head_dim, page_size, dtype);
  if (rc) return rc;
  if (n_seqs <= 0) return PKV_OK;
  const int32_t G = n_heads / n_kv_heads;
  SharedFn fn = page_size == 16 ? shared_fn(dtype, head_dim, G) : nullptr;
  if (!fn || !pkv_decode_fast_path(n_heads, n_kv_heads, head_dim, page_size, dtype, 1))
    return fail(PKV_ERR_INVALID, "shared pages need the fast decode path (see "
                "pkv_decode_fast_path)");
  if (!(scale > 0.f)) return fail(PKV_ERR_INVALID, "shared pages need a positive scale");
  if (!q || !out || !k_pool || !v_pool) return fail(PKV_ERR_INVALID, "null pointer argument");
  const uintptr_t al = (uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool |
                       (uintptr_t)k_new | (uintptr_t)v_new;
  if (al % 16) return fail(PKV_ERR_INVALID, "q, out, pools and new rows must be 16-byte aligned");
  const int32_t groups = n_kv_heads / heads_per_wg(n_kv_heads);
  if (!plan || n_work <= 0 || n_work % groups || plan_stride < kHdrInts + kStageMax * kItemInts)
    return fail(PKV_ERR_INVALID, "shared pages need a plan (pkv_plan_shared)");
  if (!kv_indices || !tiles || n_tiles <= 0 || n_merges <= 0 || n_merges > n_seqs || n_slots <= 0)
    return fail(PKV_ERR_INVALID, "shared pages need kv_indices, tiles, merges and partial slots");
  if ((k_new == nullptr) != (v_new == nullptr) || (k_new && !slot_mapping))
    return fail(PKV_ERR_INVALID, "a fused append needs k_new, v_new and slot_mapping");
  if ((int64_t)n_tiles * n_kv_heads + (int64_t)n_work * n_kv_heads > 0x7fffffffLL)
    return fail(PKV_ERR_INVALID, "too many tiles and pieces in one launch");
  DecodeWorkspace w;
  rc = split_workspace(workspace, workspace_bytes, n_seqs, n_slots, n_heads, n_kv_heads, head_dim,
                       &w);
  if (rc) return rc;
  const int32_t* list = tiles + (int64_t)n_tiles * kSharedItem;
  fn({q, out, k_pool, v_pool, num_blocks, kv_indices, n_kv_heads, scale * kLog2e,
      {tiles, list + (int64_t)n_merges * 4, w.part_o, w.part_ml}, n_tiles, list, n_merges, plan,
      n_work, plan_stride, k_new, v_new, slot_mapping, w, status_word, dtype}, (hipStream_t)stream);
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

static_assert(sizeof(pkv_shared) == 112, "the layout the Python binding fills");

extern "C" int pkv_attend_shared_batch(const void* batch, const void* q, void* out, void* k_pool,
                                       void* v_pool, float scale, const void* k_new,
                                       const void* v_new, void* stream) {
  if (!batch) return fail(PKV_ERR_INVALID, "null batch");
  const pkv_shared& b = *static_cast<const pkv_shared*>(batch);
  return pkv_attend_shared(q, out, k_pool, v_pool, b.num_blocks, b.kv_indices, b.n_seqs, b.n_heads,
                           b.n_kv_heads, b.head_dim, b.page_size, scale, b.dtype, b.tiles,
                           b.n_tiles, b.n_merges, b.plan, b.n_work, b.n_slots, b.plan_stride,
                           k_new, v_new, k_new ? b.slot_mapping : nullptr, b.workspace,
                           b.workspace_bytes, b.status_word, stream);
}
