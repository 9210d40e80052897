// Decode attention over the pages chosen for each sequence and KV head
// (selection.hip): a list of page ids each, in order, the sequence's last page
// last. Only the last page may be partly filled.
#include <algorithm>
#include <exception>
#include <vector>

#include "decode_stream.h"

namespace pkv {

int check_geometry(int32_t Hq, int32_t Hkv, int32_t D, int32_t ps, int32_t dtype);
int split_workspace(void* workspace, int64_t workspace_bytes, int32_t n_seqs, int32_t n_slots,
                    int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, DecodeWorkspace* w);

// Waves a SIMD the kernel is compiled for: the merge's registers grow with G.
template <int G> constexpr int kSelectedWaves = G <= 4 ? 4 : G == 8 ? 3 : 2;

// The piece kernel (decode_piece.h) over chosen pages: a workgroup a piece and
// KV head, heads first, so that a head's workgroups meet one L2.
template <typename T, int D, int G>
__global__ __launch_bounds__(256, kSelectedWaves<G>) void selected_kernel(
    const T* __restrict__ q, T* __restrict__ out, T* __restrict__ kpool, T* __restrict__ vpool,
    int64_t num_blocks, int32_t n_kv_heads, float scale_log2, Chosen ch, DecodeWorkspace w,
    int32_t* status) {
  __shared__ __align__(16) unsigned char smem[PieceLds<T, D, G, kChosenChunk>::BYTES];
  const int bin = blockIdx.x / n_kv_heads;
  decode_piece<T, D, G, true>(smem, blockIdx.x - bin * n_kv_heads, bin, q, out, kpool, vpool,
                              num_blocks, nullptr, 0, n_kv_heads, scale_log2, nullptr, nullptr,
                              nullptr, w.part_o, w.part_ml, w.o_bytes, w.ml_bytes, w.counters,
                              status, ch);
}

// Larger batches: the streaming decode kernel over a plan of the chosen lists,
// each KV head's page words its own.
template <typename T, int D, int G>
__global__ __launch_bounds__(kMaxWaves * 64) void selected_stream_kernel(
    const T* __restrict__ q, T* __restrict__ out, T* __restrict__ kpool, T* __restrict__ vpool,
    int64_t num_blocks, const int32_t* __restrict__ plan, int32_t stride, int32_t n_kv_heads,
    float scale_log2, DecodeWorkspace w, int32_t* status, const int32_t* __restrict__ words,
    int64_t head_words) {
  extern __shared__ __align__(16) unsigned char smem[];
  decode_stream<T, D, G, true>(smem, blockIdx.y, blockIdx.x, q, out, kpool, vpool, num_blocks,
                               plan, stride, n_kv_heads, scale_log2, nullptr, nullptr, nullptr,
                               w.part_o, w.part_ml, w.o_bytes, w.ml_bytes, w.counters, status,
                               words, head_words);
}

// Any geometry: one wave a query head, three passes over the chosen pages' keys
// (maximum, sum, weighted values), as the generic kernel does over all of them;
// probabilities stay in 32 bits, as the products with them are.
template <typename T>
__global__ __launch_bounds__(64) void selected_generic_kernel(
    const T* __restrict__ q, T* __restrict__ out, const T* __restrict__ kpool,
    const T* __restrict__ vpool, int64_t num_blocks, const int32_t* __restrict__ kv_lens,
    const int32_t* __restrict__ ids, int32_t width, int32_t pages, int32_t n_heads,
    int32_t n_kv_heads, int32_t D, int32_t ps, float scale, int32_t* status) {
  __shared__ float qs[256];
  __shared__ float pw[64];
  const int lane = threadIdx.x;
  const int seq = blockIdx.y, hq = blockIdx.x;
  const int h = hq / (n_heads / n_kv_heads);
  const int kv_len = kv_lens[seq], np = (kv_len + ps - 1) / ps;
  const int n_keys = (min(np, pages) - 1) * ps + kv_len - (np - 1) * ps;
  const int32_t* list = ids + ((int64_t)seq * n_kv_heads + h) * width;
  const int64_t row = (int64_t)n_kv_heads * D;
  for (int e = lane; e < D; e += 64)
    qs[e] = Elem<T>::to_f(q[((int64_t)seq * n_heads + hq) * D + e]);
  __syncthreads();
  auto key_row = [&](int key, const T* pool) -> const T* {
    int64_t page = list[key / ps];
    if (page < 0 || page >= num_blocks) { flag(status, PKV_STATUS_BAD_PAGE); page = 0; }
    return pool + (page * ps + key % ps) * row + (int64_t)h * D;
  };
  auto score = [&](int key) -> float {
    const T* kr = key_row(key, kpool);
    float s = 0.f;
    for (int e = 0; e < D; ++e) s += qs[e] * Elem<T>::to_f(kr[e]);
    return s * scale;
  };
  float m = -INFINITY;
  for (int key = lane; key < n_keys; key += 64) m = fmaxf(m, score(key));
  m = wave_max(m);
  float l = 0.f;
  for (int key = lane; key < n_keys; key += 64) l += expf(score(key) - m);
  const float inv = 1.f / wave_sum(l);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < n_keys; k0 += 64) {
    const int key = k0 + lane;
    float p = 0.f;
    if (key < n_keys) p = expf(score(key) - m) * inv;
    __syncthreads();
    pw[lane] = p;
    __syncthreads();
    const int nk = min(64, n_keys - k0);
    for (int u = 0; u < nk; ++u) {
      const T* vr = key_row(k0 + u, vpool);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int e = lane + 64 * c;
        if (e < D) acc[c] += pw[u] * Elem<T>::to_f(vr[e]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int e = lane + 64 * c;
    if (e < D) out[((int64_t)seq * n_heads + hq) * D + e] = Elem<T>::from_f(acc[c]);
  }
}


struct SelectedArgs {
  const void* q; void* out; void* kp; void* vp; int64_t nb; int32_t Hkv; float sl2;
  Chosen ch; DecodeWorkspace w; int32_t* status;
  const int32_t* plan; const int32_t* words; int64_t head_words; int32_t n_work, stride;
};

template <typename T, int D, int G>
static void launch_selected(const SelectedArgs& a, hipStream_t s) {
  if (a.plan) {
    const int hgw = heads_per_wg(a.Hkv), groups = a.Hkv / hgw;
    hipLaunchKernelGGL((selected_stream_kernel<T, D, G>),
                       dim3((unsigned)groups, (unsigned)(a.n_work / groups)), dim3(hgw * 64),
                       (decode_lds_bytes<T, D, G>(hgw)), s, (const T*)a.q, (T*)a.out, (T*)a.kp,
                       (T*)a.vp, a.nb, a.plan, a.stride, a.Hkv, a.sl2, a.w, a.status, a.words,
                       a.head_words);
    return;
  }
  const unsigned blocks = (unsigned)(a.ch.n_seqs * a.ch.max_parts * a.Hkv);
  hipLaunchKernelGGL((selected_kernel<T, D, G>), dim3(blocks), dim3(256), 0, s, (const T*)a.q,
                     (T*)a.out, (T*)a.kp, (T*)a.vp, a.nb, a.Hkv, a.sl2, a.ch, a.w, a.status);
}

typedef void (*SelectedFn)(const SelectedArgs&, hipStream_t);

template <typename T, int D>
static SelectedFn selected_g(int G) {
  switch (G) {
    case 1: return launch_selected<T, D, 1>;
    case 2: return launch_selected<T, D, 2>;
    case 4: return launch_selected<T, D, 4>;
    case 8: return launch_selected<T, D, 8>;
    case 16: return launch_selected<T, D, 16>;
    default: return nullptr;
  }
}

static SelectedFn selected_fn(int32_t dtype, int32_t D, int32_t G, int32_t page_size,
                              int64_t num_blocks) {
  if (page_size != 16 || num_blocks > (1LL << kPageIdBits)) return nullptr;
  if (dtype == PKV_DTYPE_F16)
    return D == 64 ? selected_g<_Float16, 64>(G) : D == 128 ? selected_g<_Float16, 128>(G) : nullptr;
  if (dtype == PKV_DTYPE_BF16)
    return D == 64 ? selected_g<__bf16, 64>(G) : D == 128 ? selected_g<__bf16, 128>(G) : nullptr;
  return nullptr;
}

static int max_parts(int32_t max_pages, int32_t pages, int32_t part_pages) {
  return (std::min(max_pages, pages) + part_pages - 1) / part_pages;
}

}  // namespace pkv

using namespace pkv;

extern "C" int64_t pkv_selected_workspace_bytes(int32_t n_seqs, int32_t max_pages, int32_t pages,
                                                int32_t part_pages, int32_t n_heads,
                                                int32_t n_kv_heads, int32_t head_dim,
                                                int32_t page_size, int64_t num_blocks,
                                                int32_t dtype) {
  if (n_seqs <= 0 || max_pages <= 0 || pages <= 0 || part_pages <= 0 || n_kv_heads <= 0 ||
      n_heads <= 0 || n_heads % n_kv_heads ||
      !selected_fn(dtype, head_dim, n_heads / n_kv_heads, page_size, num_blocks))
    return 0;
  const int64_t parts = max_parts(max_pages, pages, part_pages);
  if (parts < 2) return 0;
  if (n_seqs * parts > 0x7fffffffLL) return INT64_MAX;
  return pkv_decode_workspace_bytes(n_seqs, (int32_t)(n_seqs * parts), n_heads, n_kv_heads,
                                    head_dim);
}

extern "C" int pkv_plan_selected(const int32_t* kv_lens, int32_t n_seqs, int32_t pages,
                                 int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                 int32_t dtype, int32_t part_pages, int32_t max_workgroups,
                                 int32_t* plan, int64_t plan_capacity, int64_t* plan_needed,
                                 int32_t* n_work_out, int32_t* n_slots_out,
                                 int32_t* plan_stride_out, int32_t* places,
                                 int64_t places_capacity, int64_t* places_needed) try {
  if (n_seqs <= 0 || pages <= 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads)
    return fail(PKV_ERR_INVALID, "n_seqs, pages and heads must be positive, n_heads a multiple of "
                "n_kv_heads");
  if (!selected_fn(dtype, head_dim, n_heads / n_kv_heads, 16, 1))
    return fail(PKV_ERR_INVALID, "a plan of chosen pages needs the fast decode path");
  constexpr int PS = 16;
  std::vector<int32_t> ptr(n_seqs + 1, 0), lens(n_seqs), last(n_seqs);
  for (int32_t i = 0; i < n_seqs; ++i) {
    if (kv_lens[i] < 1) return fail(PKV_ERR_INVALID, "seq %d: kv_len=%d must be >= 1", i, kv_lens[i]);
    const int32_t all = (kv_lens[i] + PS - 1) / PS, n = std::min(all, pages);
    last[i] = kv_lens[i] - (all - 1) * PS;
    lens[i] = (n - 1) * PS + last[i];
    ptr[i + 1] = ptr[i] + n;
  }
  const std::vector<int32_t> ids(ptr[n_seqs], 0);   // the device fills the page words in
  int32_t n_work = 0, n_slots = 0, stride = 0;
  int64_t need = 0;
  const int rc = pkv_plan_decode(ptr.data(), ids.data(), lens.data(), last.data(), n_seqs, PS, 1,
                                 n_kv_heads, part_pages, max_workgroups, plan, plan_capacity, &need,
                                 &n_work, &n_slots, &stride);
  if (plan_needed) *plan_needed = need;
  if (rc) return rc;
  const int64_t bins = n_work / (n_kv_heads / heads_per_wg(n_kv_heads));
  int64_t items = 0;
  for (int64_t b = 0; b < bins; ++b) items += plan[b * stride];
  if (places_needed) *places_needed = 2 * (int64_t)n_seqs + items;
  if (2 * (int64_t)n_seqs + items > places_capacity)
    return fail(PKV_ERR_CAPACITY, "places need %lld entries, capacity %lld",
                (long long)(2 * (int64_t)n_seqs + items), (long long)places_capacity);
  auto each = [&](auto&& f) {   // every item, with the position of its first word
    for (int64_t b = 0; b < bins; ++b) {
      int64_t at = b * stride + kHdrInts;
      for (int32_t j = 0; j < plan[b * stride]; ++j) {
        const int32_t* it = plan + (b + 1) * stride - (int64_t)(j + 1) * kItemInts;
        f(it, at);
        at += it[1];
      }
    }
  };
  each([&](const int32_t* it, int64_t) { places[2 * it[0] + 1] = it[4] < 0 ? 1 : it[5]; });
  int32_t first = 0;
  for (int32_t i = 0; i < n_seqs; ++i) {
    places[2 * i] = first;
    first += places[2 * i + 1];
  }
  each([&](const int32_t* it, int64_t at) {
    places[2 * (int64_t)n_seqs + places[2 * it[0]] + (it[4] < 0 ? 0 : it[4] - it[6])] = (int32_t)at;
  });
  *n_work_out = n_work;
  *n_slots_out = n_slots;
  *plan_stride_out = stride;
  return PKV_OK;
} catch (const std::exception& e) {   // (no memory for the plan: nothing leaves a C entry)
  return fail(PKV_ERR_CAPACITY, "pkv_plan_selected: %s", e.what());
}

extern "C" int pkv_attend_selected(const void* q, void* out, void* k_pool, void* v_pool,
                                   int64_t num_blocks, const int32_t* ids, const int32_t* kv_lens,
                                   int32_t n_seqs, int32_t max_pages, int32_t pages,
                                   int32_t part_pages, int32_t n_heads, int32_t n_kv_heads,
                                   int32_t head_dim, int32_t page_size, float scale, int32_t dtype,
                                   const int32_t* plan, int32_t n_work, int32_t n_slots,
                                   int32_t plan_stride, const int32_t* words, int64_t head_words,
                                   void* workspace, int64_t workspace_bytes, int32_t* status_word,
                                   void* stream) {
  int rc = check_geometry(n_heads, n_kv_heads, head_dim, page_size, dtype);
  if (rc) return rc;
  if (n_seqs < 0 || max_pages <= 0 || pages <= 0 || num_blocks <= 0)
    return fail(PKV_ERR_INVALID, "num_blocks, max_pages and pages must be positive");
  if (part_pages < 1 || part_pages > kMaxPartPages)
    return fail(PKV_ERR_INVALID, "part_pages=%d outside [1, %d]", part_pages, kMaxPartPages);
  if (n_seqs == 0) return PKV_OK;
  if (!q || !out || !k_pool || !v_pool || !(plan ? words : ids) || !kv_lens)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const int32_t width = std::min(pages, max_pages);
  hipStream_t s = (hipStream_t)stream;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool;
  SelectedFn fn = selected_fn(dtype, head_dim, n_heads / n_kv_heads, page_size, num_blocks);
  if (plan) {
    const int32_t groups = n_kv_heads / heads_per_wg(n_kv_heads);
    if (!fn || al % 16)
      return fail(PKV_ERR_INVALID, "a plan of chosen pages needs the fast decode path and 16-byte "
                  "aligned q, out and pools");
    if (n_work <= 0 || n_work % groups || n_slots < 0 || head_words < 1 ||
        plan_stride < kHdrInts + kStageMax * kItemInts)
      return fail(PKV_ERR_INVALID, "chosen pages need a whole plan (pkv_plan_selected)");
    SelectedArgs a{q, out, k_pool, v_pool, num_blocks, n_kv_heads, scale * kLog2e, {}, {},
                   status_word, plan, words, head_words, n_work, plan_stride};
    rc = split_workspace(workspace, workspace_bytes, n_seqs, n_slots, n_heads, n_kv_heads,
                         head_dim, &a.w);
    if (rc) return rc;
    fn(a, s);
    PKV_LAUNCH_CHECK();
    return PKV_OK;
  }
  if (fn && al % 16 == 0) {
    const int parts = max_parts(max_pages, pages, part_pages);
    if ((int64_t)n_seqs * parts * n_kv_heads > 0x7fffffffLL)
      return fail(PKV_ERR_INVALID, "too many pieces in one launch");
    SelectedArgs a{q, out, k_pool, v_pool, num_blocks, n_kv_heads, scale * kLog2e,
                   {ids, kv_lens, width, pages, part_pages, parts, n_seqs}, {}, status_word,
                   nullptr, nullptr, 0, 0, 0};
    rc = split_workspace(workspace, workspace_bytes, n_seqs, parts > 1 ? n_seqs * parts : 0,
                         n_heads, n_kv_heads, head_dim, &a.w);
    if (rc) return rc;
    fn(a, s);
    PKV_LAUNCH_CHECK();
    return PKV_OK;
  }
  if (n_seqs > 65535) return fail(PKV_ERR_INVALID, "one call takes up to 65535 sequences here");
  auto go = [&](auto kernel, auto type) {
    typedef decltype(type) T;
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_heads, (unsigned)n_seqs), dim3(64), 0, s,
                       (const T*)q, (T*)out, (const T*)k_pool, (const T*)v_pool, num_blocks,
                       kv_lens, ids, width, pages, n_heads, n_kv_heads, head_dim, page_size, scale,
                       status_word);
  };
  if (dtype == PKV_DTYPE_F16) go(selected_generic_kernel<_Float16>, _Float16{});
  else if (dtype == PKV_DTYPE_BF16) go(selected_generic_kernel<__bf16>, __bf16{});
  else go(selected_generic_kernel<float>, float{});
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

static_assert(sizeof(pkv_selected) == 152, "the layout the Python binding fills");

extern "C" int pkv_attend_selected_batch(const void* batch, const void* q, void* out,
                                         void* k_pool, void* v_pool, const void* lo,
                                         const void* hi, int32_t* ordinals, float scale,
                                         void* stream) {
  if (!batch) return fail(PKV_ERR_INVALID, "null batch");
  const pkv_selected& b = *static_cast<const pkv_selected*>(batch);
  const int rc = pkv_select_pages(q, lo, hi, b.num_blocks, b.kv_indptr, b.kv_indices, b.kv_lens,
                                  b.n_seqs, b.max_pages, b.pages, b.n_heads, b.n_kv_heads,
                                  b.head_dim, b.page_size, b.dtype, b.scores, b.ids, ordinals,
                                  b.words, b.places, b.head_words, b.part_pages, b.status_word,
                                  stream);
  if (rc) return rc;
  return pkv_attend_selected(q, out, k_pool, v_pool, b.num_blocks, b.ids, b.kv_lens, b.n_seqs,
                             b.max_pages, b.pages, b.part_pages, b.n_heads, b.n_kv_heads,
                             b.head_dim, b.page_size, scale, b.dtype, b.plan,
                             b.n_work, b.n_slots, b.plan_stride, b.words, b.head_words,
                             b.workspace, b.workspace_bytes, b.status_word, stream);
}
