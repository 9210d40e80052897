// Paged decode attention for gfx950 (every sequence has one query token).
// Two kernels over one plan and with one result: decode_kernel streams bins of
// pieces, decode_piece_kernel (decode_piece.h) spreads each piece of a small
// batch over a workgroup.
//
// Work decomposition (planned on the host once per batch, pkv_plan_decode):
//
//  * Pieces. A sequence of np pages is cut into pieces of part_pages pages,
//    the remainder last; a remainder shorter than both kMinTail pages and
//    half a piece is folded into the piece before it. The small remainders give the deal below pieces that
//    fill the gaps between bins (measured 2% faster than pieces of nearly
//    equal size over six batches of 256 lognormal sequences). The cut
//    depends only on that sequence's own length, so its result never
//    depends on what it is batched with: a piece's arithmetic is the same
//    wherever it runs, and the partials of a cut sequence merge in a fixed
//    order.
//  * Bins. The pieces are dealt to a fixed number of bins, longest first, each
//    to the bin with the least work so far (LPT), so every bin ends up with
//    about the same number of pages. A bin is one workgroup per group of up
//    to 4 KV heads, and the grid is only as large as what stays resident, so
//    no workgroup waits for a slot and all of them stream until about the
//    same time. In a bin, the pieces of cut sequences that are not their
//    sequence's last come first (they publish while everything streams),
//    whole sequences next, and last pieces at the end (a last piece reads
//    its sequence's arrival count when it starts and, if every other piece
//    has published, merges at its end without publishing its own).
//  * Waves. Each wave owns one KV head and runs the bin's page stream on its
//    own (no workgroup barrier anywhere): it loads its head's 128-byte slice
//    of every token row (whole cache lines, eight lanes a row) into registers
//    one page ahead of use, copies the page to its private LDS tile, and
//    reads the tile back in the matrix-core operand layouts. One page in
//    flight per wave measured faster than two or three: with 2048 waves
//    streaming, deeper prefetch only lengthens the queue at the memory
//    system (the first page lands later, and the stream is no faster).
//    Every step issues the same loads on every path (no page skipped at the
//    end of the stream, Q and new rows staged in LDS per batch of items,
//    page words read with scalar loads), so the wait for a page never waits
//    for the page issued after it.
//
// Per wave, head and page (G query heads share the KV head, G <= 16):
//  1. S^T = K Q^T with one 16x16x32 MFMA per 32 dims: the K rows (from LDS)
//     are the A operand, Q^T the B operand (column n = query head n, zero
//     beyond G). Lane (head n, group g) then holds the scores of tokens
//     4g..4g+3 of the page for head n;
//  2. online softmax in registers: mask past kv_len, running max / sum with
//     two row swaps (v_permlane16_swap, v_permlane32_swap: VALU, no LDS
//     round trip); p = 2^(s*scale*log2e - m) rounded to the pool
//     dtype -- four values per lane that are exactly the A operand of a
//     16x16x16 MFMA. The reference max m moves lazily (only when a head's
//     max grows by more than 2^8), so most pages skip the rescale of o;
//  3. PV on MFMA: ds_read_b64_tr_b16 hands each lane 4 consecutive tokens of
//     one V dim, the B operand, one read per 16 dims.
//
// Loads cover only a page's rows below kv_len (the plan carries each page's
// live row count beside its id): the tail of a sequence's last page is
// outside the buffer range and reads as zeros without a memory access.
//
// Cut sequences merge in the same launch. Each piece publishes its partial
// (o, m, l) with 16-byte buffer stores carrying the sc1 (agent coherence)
// bit, which write through the per-XCD L2, waits until they have completed
// (s_waitcnt), then bumps its (sequence, head) arrival counter. The wave that
// sees the last arrival reads the partials back with sc1 loads (never a
// stale L2 line) and writes the output; a last piece that finds every other
// piece arrived merges without publishing its own. This avoids a second
// launch and an agent-scope release fence, whose L2 write-back walks the
// whole cache.
//
// Fused append (optional): when the caller passes the step's new K/V rows,
// the wave whose piece holds a sequence's last page writes its head's slice
// of the new row to slot_mapping's slot and patches the copy it loaded, so a
// decode step costs one launch per layer instead of two. The patch is
// applied only when slot_mapping names the same slot as the page table, so
// the result is exactly "append, then attend" (the caller guarantees that no
// other sequence of the launch reads that slot).
#include <algorithm>
#include <atomic>
#include <mutex>
#include <queue>
#include <vector>

#ifdef PKV_TIMELINE
#define PKV_TIMELINE_KERNEL
#endif
#include "decode_stream.h"

namespace pkv {

template <typename T, int D, int G>
__global__ __launch_bounds__(kMaxWaves * 64) void decode_kernel(
    const T* __restrict__ q, T* __restrict__ out, T* __restrict__ kpool, T* __restrict__ vpool,
    int64_t num_blocks, const int32_t* __restrict__ plan, int32_t stride, int32_t n_kv_heads,
    float scale_log2, const T* __restrict__ k_new, const T* __restrict__ v_new,
    const int32_t* __restrict__ slot_mapping, float* part_o, float* part_ml, uint32_t o_bytes,
    uint32_t ml_bytes, int32_t* counters, int32_t* status) {
  extern __shared__ __align__(16) unsigned char smem[];
  // grid (head groups, bins): the bin's plan block needs no division, so its
  // address is ready as soon as the kernel arguments are, and workgroups
  // dispatch in (bin, group) order (a bin's groups on neighbouring XCDs:
  // measured 2% faster than the two on one XCD)
  decode_stream<T, D, G>(smem, blockIdx.y, blockIdx.x, q, out, kpool, vpool, num_blocks, plan,
                         stride, n_kv_heads, scale_log2, k_new, v_new, slot_mapping, part_o,
                         part_ml, o_bytes, ml_bytes, counters, status);
}

template <typename T, int D, int G>
__global__ __launch_bounds__(256, kPieceWaves<D>) void decode_piece_kernel(
    const T* __restrict__ q, T* __restrict__ out, T* __restrict__ kpool, T* __restrict__ vpool,
    int64_t num_blocks, const int32_t* __restrict__ plan, int32_t stride, int32_t n_kv_heads,
    float scale_log2, const T* __restrict__ k_new, const T* __restrict__ v_new,
    const int32_t* __restrict__ slot_mapping, float* part_o, float* part_ml, uint32_t o_bytes,
    uint32_t ml_bytes, int32_t* counters, int32_t* status) {
  __shared__ __align__(16) unsigned char smem[PieceLds<T, D, G>::BYTES];
  decode_piece<T, D, G>(smem, blockIdx.x, blockIdx.y, q, out, kpool, vpool, num_blocks, plan,
                        stride, n_kv_heads, scale_log2, k_new, v_new, slot_mapping, part_o, part_ml,
                        o_bytes, ml_bytes, counters, status);
}

template <typename T, int D, int G>
static void launch(const void* q, void* out, void* kp, void* vp, int64_t nb,
                   const int32_t* plan, int32_t n_work, int32_t stride, int32_t Hkv, float sl2,
                   const void* kn, const void* vn, const int32_t* slots, float* po, float* pml,
                   uint32_t o_bytes, uint32_t ml_bytes, int32_t* cnt, int32_t* status,
                   hipStream_t s) {
  const int hgw = heads_per_wg(Hkv);
  const int groups = Hkv / hgw;
  auto go = [&](auto kernel, int heads, int threads, size_t lds) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)heads, (unsigned)(n_work / groups)), dim3(threads),
                       lds, s, (const T*)q, (T*)out, (T*)kp, (T*)vp, nb, plan, stride, Hkv, sl2,
                       (const T*)kn, (const T*)vn, slots, po, pml, o_bytes, ml_bytes, cnt, status);
  };
  if (few_pieces(n_work, stride, Hkv, D))
    go(decode_piece_kernel<T, D, G>, Hkv, 256, 0);
  else
    go(decode_kernel<T, D, G>, groups, hgw * 64, decode_lds_bytes<T, D, G>(hgw));
}

constexpr int kMaxDevices = 64;

int compute_units() {
  static std::atomic<int> known[kMaxDevices];   // asked once per device
  int dev = -1, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  cus = known[dev].load(std::memory_order_relaxed);
  if (cus <= 0) {
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
      return 0;
    known[dev].store(cus, std::memory_order_relaxed);
  }
  return cus;
}

// Workgroups of decode_kernel<T, D, G> that stay resident on one compute
// unit (registers and LDS), 0 on error.
template <typename T, int D, int G>
static int resident(int Hkv) {
  const int hgw = heads_per_wg(Hkv);
  int n = 0;
  const size_t lds = decode_lds_bytes<T, D, G>(hgw);
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, decode_kernel<T, D, G>, hgw * 64, lds) !=
      hipSuccess)
    return 0;
  return n;
}

typedef void (*LaunchFn)(const void*, void*, void*, void*, int64_t, const int32_t*, int32_t,
                         int32_t, int32_t, float, const void*, const void*, const int32_t*,
                         float*, float*, uint32_t, uint32_t, int32_t*, int32_t*, hipStream_t);
typedef int (*ResidentFn)(int);
struct Variant { LaunchFn launch; ResidentFn resident; };

template <typename T, int D>
static Variant pick_g(int G) {
  switch (G) {
    case 1: return {launch<T, D, 1>, resident<T, D, 1>};
    case 2: return {launch<T, D, 2>, resident<T, D, 2>};
    case 4: return {launch<T, D, 4>, resident<T, D, 4>};
    case 8: return {launch<T, D, 8>, resident<T, D, 8>};
    case 16: return {launch<T, D, 16>, resident<T, D, 16>};
    default: return {nullptr, nullptr};
  }
}

static Variant fast_variant(int32_t dtype, int32_t Hkv, int32_t D, int32_t G,
                            int32_t page_size) {
  if (page_size != 16 || Hkv < 1) return {nullptr, nullptr};
  if (dtype == PKV_DTYPE_F16) {
    if (D == 64) return pick_g<_Float16, 64>(G);
    if (D == 128) return pick_g<_Float16, 128>(G);
  } else if (dtype == PKV_DTYPE_BF16) {
    if (D == 64) return pick_g<__bf16, 64>(G);
    if (D == 128) return pick_g<__bf16, 128>(G);
  }
  return {nullptr, nullptr};
}

static LaunchFn fast_decode(int32_t dtype, int32_t Hkv, int32_t D, int32_t G,
                            int32_t page_size, int32_t pp) {
  if (pp < 1 || pp > kMaxPartPages) return nullptr;
  return fast_variant(dtype, Hkv, D, G, page_size).launch;
}

void run_decode(int32_t dtype, int32_t D, int32_t G, const void* q, void* out, void* kp, void* vp,
                int64_t nb, const int32_t* plan, int32_t n_work, int32_t stride, int32_t Hkv,
                float sl2, const void* kn, const void* vn, const int32_t* slots,
                const DecodeWorkspace& w, int32_t* status, hipStream_t s) {
  fast_variant(dtype, Hkv, D, G, 16).launch(q, out, kp, vp, nb, plan, n_work, stride, Hkv, sl2, kn,
                                            vn, slots, w.part_o, w.part_ml, w.o_bytes, w.ml_bytes,
                                            w.counters, status, s);
}

// Floats of partial output per (slot, KV head): the accumulator tile of
// ceil(G/4) groups of 4 head rows.
static int64_t part_floats(int32_t G, int32_t D) { return (int64_t)((G + 3) / 4) * 4 * D; }

// generic fallback lives in attention.hip
int generic_decode(const void* q, void* out, const void* kp, const void* vp, int64_t nb,
                   const int32_t* indptr, const int32_t* indices, const int32_t* kv_lens,
                   int32_t n_seqs, int32_t Hq, int32_t Hkv, int32_t D, int32_t ps, float scale,
                   int32_t dtype, int32_t* status, hipStream_t s);
int check_seq_pages(int32_t i, int32_t np, int32_t kv, int32_t last, int32_t ps);
int check_geometry(int32_t Hq, int32_t Hkv, int32_t D, int32_t ps, int32_t dtype);

}  // namespace pkv

using namespace pkv;

extern "C" int pkv_decode_fast_path(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                    int32_t page_size, int32_t dtype, int32_t part_pages) {
  if (n_kv_heads <= 0 || n_heads % n_kv_heads) return 0;
  return fast_decode(dtype, n_kv_heads, head_dim, n_heads / n_kv_heads, page_size, part_pages)
             ? 1 : 0;
}

extern "C" int pkv_decode_workgroups(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                     int32_t dtype, int32_t per_cu) {
  if (n_kv_heads <= 0 || n_heads % n_kv_heads || per_cu <= 0) return 0;
  const Variant v = fast_variant(dtype, n_kv_heads, head_dim, n_heads / n_kv_heads, 16);
  if (!v.resident) return 0;
  const int cus = compute_units();
  if (cus <= 0) return 0;
  const int fit = v.resident(n_kv_heads);
  return cus * std::min(per_cu, fit);
}

extern "C" int pkv_plan_decode(const int32_t* kv_indptr, const int32_t* kv_indices,
                               const int32_t* kv_lens, const int32_t* kv_last_page_len,
                               int32_t n_seqs, int32_t page_size, int64_t num_blocks,
                               int32_t n_kv_heads, int32_t part_pages, int32_t max_workgroups,
                               int32_t* plan, int64_t plan_capacity, int64_t* plan_needed,
                               int32_t* n_work_out, int32_t* n_slots_out,
                               int32_t* plan_stride_out) {
  if (n_seqs <= 0 || page_size <= 0 || part_pages <= 0 || part_pages > kMaxPartPages)
    return fail(PKV_ERR_INVALID, "n_seqs and page_size must be positive and part_pages in "
                "[1, %d]", kMaxPartPages);
  if (page_size > 16)
    return fail(PKV_ERR_INVALID, "page_size=%d: the decode plan holds at most 16 rows a page",
                page_size);
  if (n_kv_heads <= 0 || max_workgroups <= 0)
    return fail(PKV_ERR_INVALID, "n_kv_heads and max_workgroups must be positive");
  if (num_blocks <= 0 || num_blocks > (1LL << kPageIdBits))
    return fail(PKV_ERR_INVALID, "num_blocks=%lld outside [1, 2^%d] (decode plan page words)",
                (long long)num_blocks, kPageIdBits);
  if (kv_indptr[0] != 0) return fail(PKV_ERR_INVALID, "kv_indptr must start at 0");
  // Pieces of every sequence (part_pages pages each, the remainder last,
  // folded into the piece before it when shorter than both kMinTail and half
  // a piece), and slots
  // for cut sequences. Role: 0 a cut sequence's piece before its last, 1 a
  // whole sequence, 2 a cut sequence's last piece (it merges).
  struct Item { int32_t seq, first, np, slot, nparts, slot0, role; int64_t cost; };
  std::vector<Item> items;
  items.reserve(n_seqs);
  int32_t slots = 0;
  for (int32_t i = 0; i < n_seqs; ++i) {
    const int32_t np = kv_indptr[i + 1] - kv_indptr[i];
    int rc = check_seq_pages(i, np, kv_lens[i], kv_last_page_len[i], page_size);
    if (rc) return rc;
    const int32_t full = np / part_pages, rem = np % part_pages;
    const bool fold = full > 0 && rem > 0 && rem < std::min(kMinTail, (part_pages + 1) / 2);
    const int32_t k = full + (rem > 0 && !fold ? 1 : 0);
    int32_t first = 0;
    for (int32_t p = 0; p < k; ++p) {
      const int32_t m = p < full ? part_pages + (fold && p + 1 == full ? rem : 0) : rem;
      const int32_t role = k == 1 ? 1 : p + 1 == k ? 2 : 0;
      // cost in 1/16 pages: the pages, a start-up per piece (Q, output) and,
      // for a last piece, the merge it runs at the end of its bin
      const int64_t cost = (int64_t)m * 16 + 4 + (role == 2 ? 40 : 0);
      items.push_back({i, first, m, k > 1 ? slots + p : -1, k, k > 1 ? slots : -1, role, cost});
      first += m;
    }
    if (k > 1) slots += k;
  }
  const int hgw = heads_per_wg(n_kv_heads);
  const int n_groups = n_kv_heads / hgw;
  int64_t bins = std::max<int64_t>(1, max_workgroups / n_groups);
  bins = std::min<int64_t>(bins, (int64_t)items.size());
  // A cut piece at least half a bin long usually ends its bin, so the
  // publish / count / merge chain after its last page adds to that bin's
  // time instead of overlapping the next piece's pages: it is charged 72
  // (4.5 pages) instead of the last piece's 40 (measured on the batch-256
  // decode step: 1.4% faster; no change where bins hold many pieces).
  {
    int64_t total = 0;
    for (const Item& x : items) total += (int64_t)x.np * 16;
    const int64_t half_bin = total / bins / 2;
    for (Item& x : items)
      if (x.role != 1 && (int64_t)x.np * 16 >= half_bin) x.cost = (int64_t)x.np * 16 + 4 + 72;
  }
  // longest-processing-time-first deal into the least-loaded bin
  std::vector<int32_t> order(items.size());
  for (size_t i = 0; i < order.size(); ++i) order[i] = (int32_t)i;
  std::stable_sort(order.begin(), order.end(),
                   [&](int32_t a, int32_t b) { return items[a].cost > items[b].cost; });
  typedef std::pair<int64_t, int32_t> Load;  // (work, bin)
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> heap;
  for (int32_t b = 0; b < bins; ++b) heap.push({0, b});
  // (flat arrays: the bin of every item in dealing order, then the items of
  // each bin gathered by a counting sort, so planning allocates nothing per bin)
  const size_t n_items = items.size();
  std::vector<int32_t> bin_of(n_items), bin_count((size_t)bins + 1, 0);
  std::vector<int64_t> bin_pages((size_t)bins, 0);
  for (int32_t ix : order) {
    Load l = heap.top();
    heap.pop();
    bin_of[ix] = l.second;
    ++bin_count[l.second + 1];
    bin_pages[l.second] += items[ix].np;
    heap.push({l.first + items[ix].cost, l.second});
  }
  int64_t stride = kHdrInts + kStageMax * kItemInts;
  for (int64_t b = 0; b < bins; ++b)
    stride = std::max<int64_t>(stride, kHdrInts + ((bin_pages[b] + 3) & ~3LL) +
                                           kItemInts * (int64_t)bin_count[b + 1]);
  // (it was a multiple of 4: which one says what few_pieces asks)
  if ((stride % 8 == 0) != (bins == (int64_t)n_items)) stride += 4;
  // in a bin: pieces before a cut sequence's last, whole sequences, then last
  // pieces, each in dealing order (longest first): a stable sort by (bin, role)
  for (int64_t b = 0; b < bins; ++b) bin_count[b + 1] += bin_count[b];
  std::vector<int32_t> by_bin(n_items);
  {
    std::vector<int32_t> fill(bin_count.begin(), bin_count.end() - 1);
    for (int role = 0; role < 3; ++role)
      for (int32_t ix : order)
        if (items[ix].role == role) by_bin[fill[bin_of[ix]]++] = ix;
  }
  const int64_t need = bins * stride + kPlanTail;
  if (plan_needed) *plan_needed = need;
  if (stride > 0x7fffffff || need > plan_capacity)
    return fail(PKV_ERR_CAPACITY, "decode plan needs %lld entries, capacity %lld",
                (long long)need, (long long)plan_capacity);
  std::fill(plan, plan + need, 0);
  for (int64_t b = 0; b < bins; ++b) {
    int32_t* bp = plan + b * stride;
    bp[0] = bin_count[b + 1] - bin_count[b];
    bp[1] = (int32_t)bin_pages[b];
    int32_t* w = bp + kHdrInts;
    for (int32_t j = bin_count[b]; j < bin_count[b + 1]; ++j) {
      int32_t* it = bp + stride - (int64_t)(j - bin_count[b] + 1) * kItemInts;
      const Item& x = items[by_bin[j]];
      const int32_t np_seq = kv_indptr[x.seq + 1] - kv_indptr[x.seq];
      for (int32_t t = 0; t < x.np; ++t) {
        const int32_t pg = x.first + t;
        const int32_t id = kv_indices[kv_indptr[x.seq] + pg];
        const bool bad = id < 0 || (int64_t)id >= num_blocks;
        const int32_t live = pg == np_seq - 1 ? kv_last_page_len[x.seq] : page_size;
        *w++ = (int32_t)((uint32_t)(bad ? 0 : id) | ((uint32_t)(live - 1) << kPageIdBits) |
                         (bad ? 0x80000000u : 0u));
      }
      const bool last = x.first + x.np == np_seq;
      const int32_t vals[kItemInts] = {x.seq, x.np, x.first * page_size, kv_lens[x.seq],
                                       x.slot, x.nparts, x.slot0,
                                       (x.seq << kRowShift) | (last ? kItemLast : 0)};
      for (int k = 0; k < kItemInts; ++k) *it++ = vals[k];
    }
  }
  *n_work_out = (int32_t)(bins * n_groups);
  *n_slots_out = slots;
  *plan_stride_out = (int32_t)stride;
  return PKV_OK;
}

// Workspace: the arrival counters (n_seqs x n_kv_heads, padded to 256 bytes),
// then the partial outputs and the (m, l) pairs. Every counter is zero
// before a launch and after it.
static int64_t counter_bytes(int32_t n_seqs, int32_t n_kv_heads) {
  return ((int64_t)n_seqs * n_kv_heads * 4 + 255) / 256 * 256;
}

extern "C" int64_t pkv_decode_workspace_bytes(int32_t n_seqs, int32_t n_slots,
                                              int32_t n_heads, int32_t n_kv_heads,
                                              int32_t head_dim) {
  if (n_seqs <= 0 || n_kv_heads <= 0 || n_slots <= 0 || n_heads <= 0) return 0;
  if (n_heads % n_kv_heads) return 0;
  const int64_t po = (int64_t)n_slots * n_kv_heads * part_floats(n_heads / n_kv_heads, head_dim);
  return counter_bytes(n_seqs, n_kv_heads) + (po + (int64_t)n_slots * n_heads * 2) * 4;
}

namespace pkv {

// The parts of a decode workspace (all null when no sequence is cut):
// [arrival counters, n_seqs * n_kv_heads | partial outputs
//  [n_slots][Hkv][part_floats] | (m, l) [n_slots][Hq][2]]
int split_workspace(void* workspace, int64_t workspace_bytes, int32_t n_seqs, int32_t n_slots,
                    int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, DecodeWorkspace* w) {
  *w = DecodeWorkspace{nullptr, nullptr, nullptr, 0, 0};
  if (n_slots <= 0) return PKV_OK;
  const int64_t need = pkv_decode_workspace_bytes(n_seqs, n_slots, n_heads, n_kv_heads, head_dim);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
    return fail(PKV_ERR_CAPACITY, "split-K plan needs %lld 256-byte-aligned workspace "
                "bytes, got %lld", (long long)need, (long long)workspace_bytes);
  const int64_t pf = (int64_t)n_slots * n_kv_heads * part_floats(n_heads / n_kv_heads, head_dim);
  const int64_t mlf = (int64_t)n_slots * n_heads * 2;
  if ((pf + mlf) * 4 > 0x7fffffffLL)
    return fail(PKV_ERR_INVALID, "split-K partials exceed 2 GiB; use larger partitions");
  w->counters = (int32_t*)workspace;
  w->part_o = (float*)((char*)workspace + counter_bytes(n_seqs, n_kv_heads));
  w->part_ml = w->part_o + pf;
  w->o_bytes = (uint32_t)(pf * 4);
  w->ml_bytes = (uint32_t)(mlf * 4);
  return PKV_OK;
}

// The decode launch shared by both entry points. `zero_counters` clears the
// arrival counters at the front of the workspace with a fill kernel first
// (kept to a kernel, not a memset, so the call can sit inside a captured
// graph).
__global__ void zero_words(int32_t* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) p[i] = 0;
}

static int attend_decode(const void* q, void* out, void* k_pool, void* v_pool,
                         int64_t num_blocks, const int32_t* kv_indptr,
                         const int32_t* kv_indices, const int32_t* kv_lens, int32_t n_seqs,
                         int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                         int32_t page_size, float scale, int32_t dtype, const int32_t* plan,
                         int32_t n_work, int32_t n_slots, int32_t plan_stride,
                         const void* k_new, const void* v_new, const int32_t* slot_mapping,
                         void* workspace, int64_t workspace_bytes, bool zero_counters,
                         int32_t* status_word, void* stream) {
  int rc = check_geometry(n_heads, n_kv_heads, head_dim, page_size, dtype);
  if (rc) return rc;
  if (n_seqs <= 0) return PKV_OK;
  hipStream_t s = (hipStream_t)stream;
  const int32_t G = n_heads / n_kv_heads;
  LaunchFn fn = fast_decode(dtype, n_kv_heads, head_dim, G, page_size, 1);
  if (!fn) {
    if (k_new)
      return fail(PKV_ERR_INVALID, "a fused append needs the fast decode path "
                                   "(see pkv_decode_fast_path)");
    return generic_decode(q, out, k_pool, v_pool, num_blocks, kv_indptr, kv_indices, kv_lens,
                          n_seqs, n_heads, n_kv_heads, head_dim, page_size, scale, dtype,
                          status_word, s);
  }
  if (!plan || n_work <= 0 || n_slots < 0 || plan_stride < kHdrInts + kStageMax * kItemInts)
    return fail(PKV_ERR_INVALID, "decode needs a plan (pkv_plan_decode)");
  if (n_work % (n_kv_heads / heads_per_wg(n_kv_heads)))
    return fail(PKV_ERR_INVALID, "n_work=%d is not a whole number of bins", n_work);
  if ((k_new == nullptr) != (v_new == nullptr) || (k_new && !slot_mapping))
    return fail(PKV_ERR_INVALID, "a fused append needs k_new, v_new and slot_mapping");
  const uintptr_t al = (uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool |
                       (uintptr_t)k_new | (uintptr_t)v_new;
  if (al % 16) return fail(PKV_ERR_INVALID, "q, out, pools and new rows must be 16-byte aligned");
  DecodeWorkspace w;
  rc = split_workspace(workspace, workspace_bytes, n_seqs, n_slots, n_heads, n_kv_heads, head_dim,
                       &w);
  if (rc) return rc;
  if (w.counters && zero_counters) {
    const int64_t words = counter_bytes(n_seqs, n_kv_heads) / 4;
    hipLaunchKernelGGL(zero_words, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, s,
                       w.counters, words);
    PKV_LAUNCH_CHECK();
  }
  fn(q, out, k_pool, v_pool, num_blocks, plan, n_work, plan_stride, n_kv_heads, scale * kLog2e,
     k_new, v_new, slot_mapping, w.part_o, w.part_ml, w.o_bytes, w.ml_bytes, w.counters,
     status_word, s);
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

// Workspace of the no-allocation entry point: one file-scope device array,
// which every GPU the library runs on holds (at its own address) until the
// process ends. In host code `scratch` names a host-side stand-in, never the
// device memory: the device address is looked up once per device with
// hipGetSymbolAddress and only that address is passed to kernels.
static __device__ __align__(256) unsigned char scratch[PKV_DECODE_SCRATCH_BYTES];

static void* g_scratch_ptr[kMaxDevices];
static std::mutex g_scratch_mu;

// This device's address of `scratch`, looked up on the first call on the
// device (with it current); nullptr with the error set on failure.
static void* scratch_on_current_device() {
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) {
    fail(PKV_ERR_HIP, "no current HIP device (or device index above %d)", kMaxDevices - 1);
    return nullptr;
  }
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* ptr = nullptr;
    const hipError_t e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !ptr) {
      fail(PKV_ERR_HIP, "hipGetSymbolAddress(scratch) failed on device %d: %s", dev,
           hipGetErrorString(e));
      return nullptr;
    }
    g_scratch_ptr[dev] = ptr;
  }
  return g_scratch_ptr[dev];
}

}  // namespace pkv

extern "C" int pkv_attend_decode(const void* q, void* out, void* k_pool, void* v_pool,
                                 int64_t num_blocks, const int32_t* kv_indptr,
                                 const int32_t* kv_indices, const int32_t* kv_lens,
                                 int32_t n_seqs, int32_t n_heads, int32_t n_kv_heads,
                                 int32_t head_dim, int32_t page_size, float scale,
                                 int32_t dtype, const int32_t* plan, int32_t n_work,
                                 int32_t n_slots, int32_t plan_stride, const void* k_new,
                                 const void* v_new, const int32_t* slot_mapping,
                                 void* workspace, int64_t workspace_bytes,
                                 int32_t* status_word, void* stream) {
  return attend_decode(q, out, k_pool, v_pool, num_blocks, kv_indptr, kv_indices, kv_lens,
                       n_seqs, n_heads, n_kv_heads, head_dim, page_size, scale, dtype, plan,
                       n_work, n_slots, plan_stride, k_new, v_new, slot_mapping, workspace,
                       workspace_bytes, false, status_word, stream);
}

extern "C" int pkv_attend_decode_noalloc(const void* q, void* out, void* k_pool, void* v_pool,
                                         int64_t num_blocks, const int32_t* kv_indptr,
                                         const int32_t* kv_indices, const int32_t* kv_lens,
                                         int32_t n_seqs, int32_t n_heads, int32_t n_kv_heads,
                                         int32_t head_dim, int32_t page_size, float scale,
                                         int32_t dtype, const int32_t* plan, int32_t n_work,
                                         int32_t n_slots, int32_t plan_stride,
                                         const void* k_new, const void* v_new,
                                         const int32_t* slot_mapping, int32_t* status_word,
                                         void* stream) {
  void* ws = nullptr;
  if (n_slots > 0) {
    const int64_t need =
        pkv_decode_workspace_bytes(n_seqs, n_slots, n_heads, n_kv_heads, head_dim);
    if (need <= 0)
      return fail(PKV_ERR_INVALID, "invalid geometry for a split-K plan");
    if (need > (int64_t)PKV_DECODE_SCRATCH_BYTES)
      return fail(PKV_ERR_CAPACITY, "split-K plan needs %lld workspace bytes; the "
                  "no-allocation entry point holds at most %lld (use pkv_attend_decode with a "
                  "workspace, or larger partitions)", (long long)need,
                  (long long)PKV_DECODE_SCRATCH_BYTES);
    ws = scratch_on_current_device();
    if (!ws) return PKV_ERR_HIP;
  }
  return attend_decode(q, out, k_pool, v_pool, num_blocks, kv_indptr, kv_indices, kv_lens,
                       n_seqs, n_heads, n_kv_heads, head_dim, page_size, scale, dtype, plan,
                       n_work, n_slots, plan_stride, k_new, v_new, slot_mapping, ws,
                       (int64_t)PKV_DECODE_SCRATCH_BYTES, true, status_word, stream);
}

#ifdef PKV_TIMELINE
// Copies the instrumented build's per-wave decode timeline (the last launch
// that wrote each record) to host memory: at most `bytes` bytes.
extern "C" int pkv_timeline_read(void* host, int64_t bytes) {
  if (bytes > (int64_t)sizeof(pkv::pkv_timeline)) bytes = sizeof(pkv::pkv_timeline);
  return hipMemcpyFromSymbol(host, HIP_SYMBOL(pkv::pkv_timeline), (size_t)bytes, 0,
                             hipMemcpyDeviceToHost) == hipSuccess ? 0 : -1;
}
#endif
