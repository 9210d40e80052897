// Attention over selected pages: for long histories, each query reads only the
// pages whose keys can score high.
//
//  * page_bounds_kernel keeps, per page and KV head, the elementwise minimum
//    and maximum of the page's keys (exact, in the pool dtype).
//  * score_kernel bounds a page's scores from them: for query head g of KV
//    head h, q_g . k <= sum_d q_gd * (q_gd < 0 ? lo_d : hi_d) for every key k of
//    the page; the page's score is the largest over the KV head's query heads.
//    Sums run in 64 bits: which page is in and which is out must not hang on
//    the order of a sum.
//  * select_kernel takes a sequence's last page and the best of the others
//    (equal scores: the lower page; a NaN beats every number), in page order.
//  * the attention then runs over the chosen pages (attend_selected).
#include <algorithm>

#include "mfma.h"

namespace pkv {

int check_geometry(int32_t Hq, int32_t Hkv, int32_t D, int32_t ps, int32_t dtype);

// ------------------------------------------------------------- page bounds ---
// One workgroup a page and layer, one vector of V elements of the page's rows a
// thread at a time, all rows of the page in a row. A NaN stays: it bounds nothing.
template <typename T, int V>
__global__ __launch_bounds__(256) void page_bounds_kernel(
    const char* __restrict__ k_pool, int64_t pool_step, char* __restrict__ lo,
    char* __restrict__ hi, int64_t bounds_step, int64_t num_blocks,
    const int32_t* __restrict__ ids, int32_t page_size, int32_t row_vecs, int32_t* status) {
  typedef T vec __attribute__((ext_vector_type(V)));
  const int64_t id = ids ? ids[blockIdx.x] : (int64_t)blockIdx.x;
  if (id < 0 || id >= num_blocks) {
    if (threadIdx.x == 0 && blockIdx.y == 0) flag(status, PKV_STATUS_BAD_BLOCK);
    return;
  }
  const int64_t layer = blockIdx.y;
  const vec* src = reinterpret_cast<const vec*>(k_pool + layer * pool_step) +
                   id * page_size * row_vecs;
  for (int c = threadIdx.x; c < row_vecs; c += blockDim.x) {
    vec mn = src[c], mx = mn;
#pragma unroll 16
    for (int r = 1; r < page_size; ++r) {
      const vec x = src[(int64_t)r * row_vecs + c];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float e = Elem<T>::to_f(x[i]);
        const bool nan = e != e;
        if (nan || e < Elem<T>::to_f(mn[i])) mn[i] = x[i];
        if (nan || e > Elem<T>::to_f(mx[i])) mx[i] = x[i];
      }
    }
    reinterpret_cast<vec*>(lo + layer * bounds_step)[id * row_vecs + c] = mn;
    reinterpret_cast<vec*>(hi + layer * bounds_step)[id * row_vecs + c] = mx;
  }
}

// Pages of a sequence, within its page list and the room for its scores.
__device__ __forceinline__ int seq_pages(const int32_t* kv_indptr, const int32_t* kv_lens, int seq,
                                         int page_size, int64_t room) {
  const int np = (kv_lens[seq] + page_size - 1) / page_size;
  return (int)min((int64_t)min(np, kv_indptr[seq + 1] - kv_indptr[seq]), room);
}

// ------------------------------------------------------------------- scores ---
// One wave a KV head and 64 pages, a page a lane: the lane reads its page's two
// rows of bounds, q is the same for the whole wave.
template <typename T, int V>
__global__ __launch_bounds__(64) void score_kernel(
    const T* __restrict__ q, const T* __restrict__ lo, const T* __restrict__ hi,
    int64_t num_blocks, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, const int32_t* __restrict__ kv_lens, int32_t n_heads,
    int32_t n_kv_heads, int32_t D, int32_t page_size, int32_t pages, int64_t stride,
    double* __restrict__ scores, int32_t* status) {
  typedef T vec __attribute__((ext_vector_type(V)));
  const int seq = blockIdx.z, h = blockIdx.y;
  const int np = seq_pages(kv_indptr, kv_lens, seq, page_size, stride);
  const int p = blockIdx.x * 64 + threadIdx.x;
  if (np <= pages || p >= np - 1) return;   // nothing to choose; the last page is in
  int64_t id = kv_indices[kv_indptr[seq] + p];
  if (id < 0 || id >= num_blocks) {
    flag(status, PKV_STATUS_BAD_PAGE);
    id = 0;
  }
  const int G = n_heads / n_kv_heads;
  const int64_t at = (id * n_kv_heads + h) * D;
  double best = 0;
  for (int g = 0; g < G; ++g) {
    const T* qr = q + ((int64_t)seq * n_heads + h * G + g) * D;
    double s = 0;
    for (int d = 0; d < D; d += V) {
      const vec a = *reinterpret_cast<const vec*>(lo + at + d);
      const vec b = *reinterpret_cast<const vec*>(hi + at + d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float x = Elem<T>::to_f(qr[d + i]);
        s = __builtin_fma((double)x, (double)Elem<T>::to_f(x < 0.f ? a[i] : b[i]), s);
      }
    }
    best = g == 0 || s > best || s != s ? s : best;
  }
  scores[((int64_t)seq * n_kv_heads + h) * stride + p] = best;
}

// ------------------------------------------------------------------- choice ---
// A score as an unsigned number of the same order, a NaN above every number.
__device__ __forceinline__ uint64_t order_of(double s) {
  if (s != s) return ~0ull;
  const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0);   // -0 + 0 = 0
  return u >> 63 ? ~u : u | 1ull << 63;
}

// One workgroup of 256 threads a sequence and KV head. The k-th largest order
// value is found 8 bits at a time from a histogram of the values that agree
// with the bits found so far; then pages above it, and the first of those equal
// to it, are taken in page order.
__global__ __launch_bounds__(256) void select_kernel(
    const double* __restrict__ scores, int64_t stride, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, const int32_t* __restrict__ kv_lens,
    int32_t n_kv_heads, int32_t page_size, int32_t pages, int32_t width,
    int32_t* __restrict__ ids, int32_t* __restrict__ ordinals) {
  __shared__ int32_t hist[256], tails[256];
  __shared__ uint64_t found;
  __shared__ int32_t need;
  const int seq = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
  const int np = seq_pages(kv_indptr, kv_lens, seq, page_size, stride);
  const int32_t* table = kv_indices + kv_indptr[seq];
  const int64_t row = ((int64_t)seq * n_kv_heads + h) * width;
  auto put = [&](int j, int p) {
    ids[row + j] = table[p];
    ordinals[row + j] = p;
  };
  if (np <= pages) {
    for (int j = tid; j < width; j += 256) {
      if (j < np) put(j, j);
      else { ids[row + j] = -1; ordinals[row + j] = -1; }
    }
    return;
  }
  const int n = np - 1, k = pages - 1;
  if (tid == 0) put(k, n);    // (pages <= width here)
  if (k == 0) return;
  const double* sc = scores + ((int64_t)seq * n_kv_heads + h) * stride;
  if (tid == 0) { found = 0; need = k; }
  for (int shift = 56; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    const uint64_t prefix = found;
    const int left = need;
    for (int p = tid; p < n; p += 256) {
      const uint64_t u = order_of(sc[p]);
      if (shift == 56 || (u >> (shift + 8)) == prefix)
        atomicAdd(&hist[(u >> shift) & 255], 1);
    }
    __syncthreads();
    // values in bins above this one
    int above = 0;
    for (int b = tid + 1; b < 256; ++b) above += hist[b];
    if (above < left && above + hist[tid] >= left) {
      found = prefix << 8 | (uint64_t)tid;
      need = left - above;
    }
    __syncthreads();
  }
  // each thread owns a run of pages, so page order is thread order
  const uint64_t limit = found;
  const int ties = need, run = (n + 255) / 256;
  const int p0 = min(n, tid * run), p1 = min(n, p0 + run);
  int above = 0, equal = 0;
  for (int p = p0; p < p1; ++p) {
    const uint64_t u = order_of(sc[p]);
    above += u > limit;
    equal += u == limit;
  }
  hist[tid] = above;
  tails[tid] = equal;
  __syncthreads();
  int a = 0, e = 0;
  for (int t = 0; t < tid; ++t) { a += hist[t]; e += tails[t]; }
  for (int p = p0; p < p1; ++p) {
    const uint64_t u = order_of(sc[p]);
    if (u > limit || (u == limit && e < ties)) put(a + min(e, ties), p);
    a += u > limit;
    e += u == limit;
  }
}

}  // namespace pkv

using namespace pkv;

extern "C" int pkv_page_bounds(const void* k_pool, int64_t pool_step, void* lo, void* hi,
                               int64_t bounds_step, int32_t n_layers, int64_t num_blocks,
                               const int32_t* ids, int64_t n_ids, int32_t n_kv_heads,
                               int32_t head_dim, int32_t page_size, int32_t dtype,
                               int32_t* status_word, void* stream) {
  int rc = check_geometry(n_kv_heads, n_kv_heads, head_dim, page_size, dtype);
  if (rc) return rc;
  if (n_layers <= 0 || n_layers > 65535 || num_blocks <= 0 || n_ids < 0 || n_ids > 0x7fffffffLL)
    return fail(PKV_ERR_INVALID, "n_layers and num_blocks must be positive, and one call takes "
                "up to 65535 layers and 2^31 - 1 pages");
  if (!ids && n_ids > num_blocks)
    return fail(PKV_ERR_INVALID, "%lld pages of a pool of %lld", (long long)n_ids,
                (long long)num_blocks);
  if (n_ids == 0) return PKV_OK;
  if (!k_pool || !lo || !hi) return fail(PKV_ERR_INVALID, "null pointer argument");
  const int64_t row = (int64_t)n_kv_heads * head_dim * elem_bytes(dtype);
  const uintptr_t at = (uintptr_t)k_pool | (uintptr_t)lo | (uintptr_t)hi | (uintptr_t)row |
                       (uintptr_t)pool_step | (uintptr_t)bounds_step;
  const int V = at % 16 ? 1 : 16 / elem_bytes(dtype);
  const int32_t vecs = (int32_t)((int64_t)n_kv_heads * head_dim / V);
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_ids, (unsigned)n_layers),
                       dim3(std::min(256, (vecs + 63) / 64 * 64)), 0, s, (const char*)k_pool,
                       pool_step, (char*)lo, (char*)hi, bounds_step, num_blocks, ids, page_size,
                       vecs, status_word);
  };
  if (dtype == PKV_DTYPE_F16)
    V == 8 ? go(page_bounds_kernel<_Float16, 8>) : go(page_bounds_kernel<_Float16, 1>);
  else if (dtype == PKV_DTYPE_BF16)
    V == 8 ? go(page_bounds_kernel<__bf16, 8>) : go(page_bounds_kernel<__bf16, 1>);
  else
    V == 4 ? go(page_bounds_kernel<float, 4>) : go(page_bounds_kernel<float, 1>);
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

extern "C" int pkv_select_pages(const void* q, const void* lo, const void* hi, int64_t num_blocks,
                                const int32_t* kv_indptr, const int32_t* kv_indices,
                                const int32_t* kv_lens, int32_t n_seqs, int32_t max_pages,
                                int32_t pages, int32_t n_heads, int32_t n_kv_heads,
                                int32_t head_dim, int32_t page_size, int32_t dtype,
                                double* scores, int32_t* ids, int32_t* ordinals,
                                int32_t* status_word, void* stream) {
  int rc = check_geometry(n_heads, n_kv_heads, head_dim, page_size, dtype);
  if (rc) return rc;
  if (n_seqs < 0 || n_seqs > 65535 || n_kv_heads > 65535 || max_pages <= 0 || pages <= 0)
    return fail(PKV_ERR_INVALID, "max_pages and pages must be positive, and one call takes up to "
                "65535 sequences and KV heads");
  if (n_seqs == 0) return PKV_OK;
  if (!q || !lo || !hi || !kv_indptr || !kv_indices || !kv_lens || !ids || !ordinals ||
      (max_pages > pages && !scores))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const int32_t width = std::min(pages, max_pages);
  hipStream_t s = (hipStream_t)stream;
  if (max_pages > pages && pages > 1) {
    const uintptr_t at = (uintptr_t)lo | (uintptr_t)hi |
                         (uintptr_t)((int64_t)head_dim * elem_bytes(dtype));
    const bool wide = at % 16 == 0;
    auto go = [&](auto kernel, auto type) {
      typedef decltype(type) T;
      hipLaunchKernelGGL(kernel, dim3((unsigned)((max_pages + 62) / 64), (unsigned)n_kv_heads,
                                      (unsigned)n_seqs),
                         dim3(64), 0, s, (const T*)q, (const T*)lo, (const T*)hi, num_blocks,
                         kv_indptr, kv_indices, kv_lens, n_heads, n_kv_heads, head_dim, page_size,
                         pages, (int64_t)max_pages, scores, status_word);
    };
    if (dtype == PKV_DTYPE_F16)
      wide ? go(score_kernel<_Float16, 8>, _Float16{}) : go(score_kernel<_Float16, 1>, _Float16{});
    else if (dtype == PKV_DTYPE_BF16)
      wide ? go(score_kernel<__bf16, 8>, __bf16{}) : go(score_kernel<__bf16, 1>, __bf16{});
    else
      wide ? go(score_kernel<float, 4>, float{}) : go(score_kernel<float, 1>, float{});
    PKV_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(select_kernel, dim3((unsigned)n_kv_heads, (unsigned)n_seqs), dim3(256), 0, s,
                     scores, (int64_t)max_pages, kv_indptr, kv_indices, kv_lens, n_kv_heads,
                     page_size, pages, width, ids, ordinals);
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}
