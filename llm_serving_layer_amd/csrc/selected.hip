// Decode attention over the pages chosen for each sequence and KV head
// (selection.hip): a list of page ids each, in order, the sequence's last page
// last. Only the last page may be partly filled.
#include <algorithm>

#include "decode_piece.h"

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

// Any geometry: one wave a query head, three passes over the chosen pages' keys
// (maximum, sum, weighted values), as the generic kernel does over all of them.
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
    if (key < n_keys) p = Elem<T>::to_f(Elem<T>::from_f(expf(score(key) - m) * inv));
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
};

template <typename T, int D, int G>
static void launch_selected(const SelectedArgs& a, hipStream_t s) {
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

extern "C" int pkv_attend_selected(const void* q, void* out, void* k_pool, void* v_pool,
                                   int64_t num_blocks, const int32_t* ids, const int32_t* kv_lens,
                                   int32_t n_seqs, int32_t max_pages, int32_t pages,
                                   int32_t part_pages, int32_t n_heads, int32_t n_kv_heads,
                                   int32_t head_dim, int32_t page_size, float scale, int32_t dtype,
                                   void* workspace, int64_t workspace_bytes, int32_t* status_word,
                                   void* stream) {
  int rc = check_geometry(n_heads, n_kv_heads, head_dim, page_size, dtype);
  if (rc) return rc;
  if (n_seqs < 0 || max_pages <= 0 || pages <= 0 || num_blocks <= 0)
    return fail(PKV_ERR_INVALID, "num_blocks, max_pages and pages must be positive");
  if (part_pages < 1 || part_pages > kMaxPartPages)
    return fail(PKV_ERR_INVALID, "part_pages=%d outside [1, %d]", part_pages, kMaxPartPages);
  if (n_seqs == 0) return PKV_OK;
  if (!q || !out || !k_pool || !v_pool || !ids || !kv_lens)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const int32_t width = std::min(pages, max_pages);
  hipStream_t s = (hipStream_t)stream;
  const uintptr_t al = (uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool;
  SelectedFn fn = selected_fn(dtype, head_dim, n_heads / n_kv_heads, page_size, num_blocks);
  if (fn && al % 16 == 0) {
    const int parts = max_parts(max_pages, pages, part_pages);
    if ((int64_t)n_seqs * parts * n_kv_heads > 0x7fffffffLL)
      return fail(PKV_ERR_INVALID, "too many pieces in one launch");
    SelectedArgs a{q, out, k_pool, v_pool, num_blocks, n_kv_heads, scale * kLog2e,
                   {ids, kv_lens, width, pages, part_pages, parts, n_seqs}, {}, status_word};
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

static_assert(sizeof(pkv_selected) == 112, "the layout the Python binding fills");

extern "C" int pkv_attend_selected_batch(const void* batch, const void* q, void* out,
                                         void* k_pool, void* v_pool, const void* lo,
                                         const void* hi, int32_t* ordinals, float scale,
                                         void* stream) {
  if (!batch) return fail(PKV_ERR_INVALID, "null batch");
  const pkv_selected& b = *static_cast<const pkv_selected*>(batch);
  const int rc = pkv_select_pages(q, lo, hi, b.num_blocks, b.kv_indptr, b.kv_indices, b.kv_lens,
                                  b.n_seqs, b.max_pages, b.pages, b.n_heads, b.n_kv_heads,
                                  b.head_dim, b.page_size, b.dtype, b.scores, b.ids, ordinals,
                                  b.status_word, stream);
  if (rc) return rc;
  return pkv_attend_selected(q, out, k_pool, v_pool, b.num_blocks, b.ids, b.kv_lens, b.n_seqs,
                             b.max_pages, b.pages, b.part_pages, b.n_heads, b.n_kv_heads,
                             b.head_dim, b.page_size, scale, b.dtype, b.workspace,
                             b.workspace_bytes, b.status_word, stream);
}
