// Attention over selected pages: for long histories, each query reads only the
// pages whose keys can score high.
//
//  * page_bounds_kernel keeps, per page and KV head, the elementwise minimum
//    and maximum of the page's keys (exact, in the pool dtype).
//  * score_kernel bounds a page's scores from them: for query head g of KV
//    head h, q_g . k <= sum_d q_gd * (q_gd < 0 ? lo_d : hi_d) for every key k of
//    the page; the page's score is the largest over the KV head's query heads.
//    A score is a sum in 64 bits: which page is in and which is out must not
//    hang on the order of a sum. 16-bit pools sum in 32 bits first, and only
//    pages whose sums lie too close to the cut for that are summed in 64.
//  * select_kernel takes a sequence's last page and the best of the others
//    (equal scores: the lower page; a NaN beats every number), in page order.
//  * the attention then runs over the chosen pages (attend_selected).
#include <algorithm>
#include <type_traits>

#include "mfma.h"

namespace pkv {

int check_geometry(int32_t Hq, int32_t Hkv, int32_t D, int32_t ps, int32_t dtype);

// ------------------------------------------------------------- page bounds ---
// One workgroup a page and layer, one vector of V elements of the page's rows a
// thread at a time, all rows of the page in a row. A NaN stays: it bounds nothing.
// PS rows a page, all of them in flight (0: page_size, one after another).
template <typename T, int V, int PS>
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
    vec mn, mx;
    auto take = [&](const vec& x) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float e = Elem<T>::to_f(x[i]);
        const bool nan = e != e;
        if (nan || e < Elem<T>::to_f(mn[i])) mn[i] = x[i];
        if (nan || e > Elem<T>::to_f(mx[i])) mx[i] = x[i];
      }
    };
    if constexpr (PS > 0) {
      vec x[PS];
#pragma unroll
      for (int r = 0; r < PS; ++r) x[r] = src[(int64_t)r * row_vecs + c];
      mn = mx = x[0];
#pragma unroll
      for (int r = 1; r < PS; ++r) take(x[r]);
    } else {
      mn = mx = src[c];
      for (int r = 1; r < page_size; ++r) take(src[(int64_t)r * row_vecs + c]);
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

// The same for head dims of 64 and 128 and 1, 2, 4, 8 or 16 query heads a KV
// head. A row of bounds is spread over D / V lanes, 16 bytes each, so loads are
// whole lines and a wave takes 64 V / D pages at a step; a lane keeps its V
// elements of up to GQ = 4 query heads in 64 bits. The bound's choice of lo or
// hi is made in 32 bits, where it is one instruction: with the conversion and
// the product that follow, 3 a query element, and 2 to unpack each element of
// lo and hi. The row's sum over its lanes halves the query heads held with the
// lanes left (each lane keeps half of what it has and adds its partner's), so
// 4 heads over 16 lanes take 5 additions, not 16. More than 4 query heads are
// split over the waves of a workgroup.
constexpr int kScoreSteps = 4;   // page groups a wave has in flight

template <int Mask> __device__ __forceinline__ double lane_xor(double v) {
  return __builtin_bit_cast(double, __shfl_xor((unsigned long long)__builtin_bit_cast(
                                                   unsigned long long, v), Mask));
}

template <typename T, int D, int G>
struct ScoreShape {
  static constexpr int V = 16 / (int)sizeof(T);
  static constexpr int L = D / V;                 // lanes a page
  static constexpr int GQ = G < 4 ? G : 4;        // query heads a wave
  static constexpr int QW = G / GQ;               // waves that share a page
  static constexpr int PW = 64 / L;               // pages of a wave's step
  static constexpr int PAGES = 4 / QW * PW * kScoreSteps;   // of a workgroup
};

// The maximum over the heads of the sums over a page's L lanes of s[0 .. N - 1],
// in every one of the page's lanes; NaN if one of them is.
template <int N, int L> __device__ __forceinline__ double head_max(const double* s) {
  auto larger = [](double a, double b) { return a != a || a > b ? a : b; };
  if constexpr (L == 1) {
    double m = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = larger(s[i], m);
    return m;
  } else if constexpr (N > 1) {
    const bool up = threadIdx.x & (L / 2);
    double t[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const double mine = up ? s[N / 2 + i] : s[i], other = up ? s[i] : s[N / 2 + i];
      t[i] = mine + lane_xor<L / 2>(other);
    }
    const double m = head_max<N / 2, L / 2>(t);
    return larger(lane_xor<L / 2>(m), m);
  } else {
    const double t[1] = {s[0] + lane_xor<L / 2>(s[0])};
    return head_max<1, L / 2>(t);
  }
}

template <typename T, int D, int G>
__global__ __launch_bounds__(256) void score_rows_kernel(
    const T* __restrict__ q, const T* __restrict__ lo, const T* __restrict__ hi,
    int64_t num_blocks, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, const int32_t* __restrict__ kv_lens,
    int32_t n_kv_heads, int32_t page_size, int32_t pages, int64_t stride,
    double* __restrict__ scores, int32_t* status) {
  typedef ScoreShape<T, D, G> S;
  constexpr int V = S::V, L = S::L, GQ = S::GQ, PW = S::PW;
  typedef T vec __attribute__((ext_vector_type(V)));
  __shared__ double part[S::QW > 1 ? 4 * PW * kScoreSteps : 1];
  const int h = blockIdx.x, seq = blockIdx.z;
  const int np = seq_pages(kv_indptr, kv_lens, seq, page_size, stride);
  const int n = np - 1;    // candidates; the last page is in
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int quad = wave % S::QW, group = wave / S::QW;
  const int first = blockIdx.y * S::PAGES + group * (PW * kScoreSteps);
  if (np <= pages || (int)blockIdx.y * S::PAGES >= n) return;
  const int32_t* table = kv_indices + kv_indptr[seq];
  const int c = lane % L;
  int64_t at[kScoreSteps];
#pragma unroll
  for (int i = 0; i < kScoreSteps; ++i) {
    const int p = first + i * PW + lane / L;
    int64_t id = table[min(p, n - 1)];
    if (id < 0 || id >= num_blocks) {
      flag(status, PKV_STATUS_BAD_PAGE);
      id = 0;
    }
    at[i] = (id * n_kv_heads + h) * D + c * V;
  }
  vec a[kScoreSteps], b[kScoreSteps];
#pragma unroll
  for (int i = 0; i < kScoreSteps; ++i) {
    a[i] = *reinterpret_cast<const vec*>(lo + at[i]);
    b[i] = *reinterpret_cast<const vec*>(hi + at[i]);
  }
  double x[GQ][V];
#pragma unroll
  for (int g = 0; g < GQ; ++g) {
    const vec t = *reinterpret_cast<const vec*>(
        q + (((int64_t)seq * n_kv_heads + h) * G + quad * GQ + g) * D + c * V);
#pragma unroll
    for (int j = 0; j < V; ++j) x[g][j] = (double)Elem<T>::to_f(t[j]);
  }
#pragma unroll
  for (int i = 0; i < kScoreSteps; ++i) {
    double s[GQ];
#pragma unroll
    for (int g = 0; g < GQ; ++g) s[g] = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float l = Elem<T>::to_f(a[i][j]), u = Elem<T>::to_f(b[i][j]);
#pragma unroll
      for (int g = 0; g < GQ; ++g)
        s[g] = __builtin_fma(x[g][j], (double)(x[g][j] < 0 ? l : u), s[g]);
    }
    double m = head_max<GQ, L>(s);
    const int p = first + i * PW + lane / L;
    if constexpr (S::QW > 1) {
      if (c == 0) part[(wave * kScoreSteps + i) * PW + lane / L] = m;
    } else {
      if (c == 0 && p < n) scores[((int64_t)seq * n_kv_heads + h) * stride + p] = m;
    }
  }
  if constexpr (S::QW > 1) {
    __syncthreads();
    constexpr int N = PW * kScoreSteps;   // pages of a group of waves
    for (int i = threadIdx.x; i < 4 / S::QW * N; i += 256) {
      const int w = i / N * S::QW, k = i % N, p = blockIdx.y * S::PAGES + i;
      double m = part[w * N + k];
#pragma unroll
      for (int j = 1; j < S::QW; ++j) {
        const double o = part[(w + j) * N + k];
        m = o != o || o > m ? o : m;
      }
      if (p < n) scores[((int64_t)seq * n_kv_heads + h) * stride + p] = m;
    }
  }
}

// 16-bit pools: the same sums in 32 bits, a product or two an instruction, lo or
// hi taken for two elements at once by q's sign bits: 1 or 1.5 instructions a
// query element instead of 3 and no unpacking, which leaves the kernel bound by
// its loads (16 sequences of 20 000 to 60 000 tokens, 8 KV heads, head_dim 128,
// bf16: 43.5 -> 30.6 us, 5.2 TB/s). near() says how far such a sum may be off; for it each workgroup also
// leaves the largest magnitude among its pages' bounds.
constexpr int kNearSteps = 4;

template <typename T, int D, int G>
struct NearShape {
  static constexpr int L = D / 8;                 // lanes a page, 8 elements each
  static constexpr int GQ = G < 4 ? G : 4;        // query heads a wave
  static constexpr int QW = G / GQ;               // waves that share a page
  static constexpr int PW = 64 / L;               // pages of a wave's step
  static constexpr int PAGES = 4 / QW * PW * kNearSteps;   // of a workgroup
};

// How far a score in 32 bits may be off: a lane's 8 products and the sums over up
// to 16 lanes are at most 12 steps (the bf16 dot2, measured over 2^20 random
// operands of sizes down to 2^-20, is off by 1.7 2^-24 of its terms' magnitudes,
// less than two roundings), together less than 16 2^-23 of sum |q| times the
// largest bound; subnormal bf16 operands (of up to D query elements, or bounds)
// and sums may be taken for zero. Infinite
// where anything is infinite or no number, or where a sum could pass the largest
// float on its way (none is larger than that product but for its roundings: from
// half of it on): then nothing is settled by the 32-bit sums.
__device__ __forceinline__ float near(float q_sum, float b_max, int D) {
  if (!(q_sum * b_max < 1.7014118e38f)) return INFINITY;
  constexpr float kTiny = 1.1754944e-38f;
  return q_sum * (b_max * (16.f * 1.1920929e-7f) + kTiny) + b_max * ((float)D * kTiny) + 1e-36f;
}

// (fp16: dot2 loses low bits of products below 2^-24 or so, a mixed fma does not)
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c, _Float16) {
  const f16x2 x = __builtin_bit_cast(f16x2, a), y = __builtin_bit_cast(f16x2, b);
  return __builtin_fmaf((float)x[1], (float)y[1], __builtin_fmaf((float)x[0], (float)y[0], c));
}
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c, __bf16) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, a), __builtin_bit_cast(b2, b), c,
                                         false);
}

template <typename T, int D, int G>
__global__ __launch_bounds__(256) void near_scores_kernel(
    const T* __restrict__ q, const T* __restrict__ lo, const T* __restrict__ hi,
    int64_t num_blocks, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, const int32_t* __restrict__ kv_lens,
    int32_t n_kv_heads, int32_t page_size, int32_t pages, int64_t stride,
    float* __restrict__ scores, int32_t* status) {
  typedef NearShape<T, D, G> S;
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  constexpr int L = S::L, GQ = S::GQ, PW = S::PW, N = PW * kNearSteps;
  __shared__ float part[S::QW > 1 ? 4 * N : 1], largest[4];
  const int h = blockIdx.x, seq = blockIdx.z;
  const int np = seq_pages(kv_indptr, kv_lens, seq, page_size, stride);
  const int n = np - 1;    // candidates; the last page is in
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int quad = wave % S::QW, group = wave / S::QW;
  const int first = blockIdx.y * S::PAGES + group * N;
  if (np <= pages || (int)blockIdx.y * S::PAGES >= n) return;
  const int32_t* table = kv_indices + kv_indptr[seq];
  const int c = lane % L;
  int64_t at[kNearSteps];
#pragma unroll
  for (int i = 0; i < kNearSteps; ++i) {
    int64_t id = table[min(first + i * PW + lane / L, n - 1)];
    if (id < 0 || id >= num_blocks) {
      flag(status, PKV_STATUS_BAD_PAGE);
      id = 0;
    }
    at[i] = (id * n_kv_heads + h) * D + c * 8;
  }
  u32x4 a[kNearSteps], b[kNearSteps];
#pragma unroll
  for (int i = 0; i < kNearSteps; ++i) {
    a[i] = *reinterpret_cast<const u32x4*>(lo + at[i]);
    b[i] = *reinterpret_cast<const u32x4*>(hi + at[i]);
  }
  u32x4 x[GQ], neg[GQ];   // q, and ones where it is below zero
#pragma unroll
  for (int g = 0; g < GQ; ++g) {
    x[g] = *reinterpret_cast<const u32x4*>(
        q + (((int64_t)seq * n_kv_heads + h) * G + quad * GQ + g) * D + c * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = x[g][j];
      neg[g][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, w) >> 15);
    }
  }
  // The largest magnitude: of lo as whole numbers (a negative one, of the largest
  // magnitude, before any positive), of hi as signed ones.
  u16x2 ml{0, 0};
  i16x2 mh{-32768, -32768};
  float out[kNearSteps];
#pragma unroll
  for (int i = 0; i < kNearSteps; ++i) {
    float s[GQ];
#pragma unroll
    for (int g = 0; g < GQ; ++g) s[g] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (as scalars: a bit cast of a vector's element takes the vector's first)
      const uint32_t wl = a[i][j], wh = b[i][j];
      ml = __builtin_elementwise_max(ml, __builtin_bit_cast(u16x2, wl));
      mh = __builtin_elementwise_max(mh, __builtin_bit_cast(i16x2, wh));
#pragma unroll
      for (int g = 0; g < GQ; ++g)
        s[g] = dot2(x[g][j], (neg[g][j] & wl) | (~neg[g][j] & wh), s[g], T{});
    }
#pragma unroll
    for (int g = 0; g < GQ; ++g) {   // over the page's L lanes
      s[g] += dpp<0xB1>(s[g]);
      s[g] += dpp<0x4E>(s[g]);
      s[g] += dpp<0x141>(s[g]);
      if (L == 16) s[g] += dpp<0x140>(s[g]);
    }
    out[i] = s[0];
#pragma unroll
    for (int g = 1; g < GQ; ++g) out[i] = fmaxf(out[i], s[g]);
  }
  // the pages' scores, then the workgroups' maxima
  float* row = scores + ((int64_t)seq * n_kv_heads + h) * 2 * stride;
  auto magnitude = [](uint32_t bits) {
    return Elem<T>::to_f(__builtin_bit_cast(T, (unsigned short)(bits & 0x7fff)));
  };
  float m = fmaxf(fmaxf(magnitude(ml[0]), magnitude(ml[1])),
                  fmaxf(magnitude((unsigned short)mh[0]), magnitude((unsigned short)mh[1])));
  // (a NaN shows: fmaxf would drop it)
  auto special = [](uint32_t bits) {
    return (bits & 0x7fff) >= (__is_same(T, _Float16) ? 0x7c00 : 0x7f80);
  };
  if (special(ml[0]) || special(ml[1]) || special((unsigned short)mh[0]) ||
      special((unsigned short)mh[1]))
    m = INFINITY;
  m = wave_max(m);
  if (lane == 0) largest[wave] = m;
  if constexpr (S::QW > 1) {
#pragma unroll
    for (int i = 0; i < kNearSteps; ++i)
      if (c == 0) part[wave * N + i * PW + lane / L] = out[i];
  } else {
#pragma unroll
    for (int i = 0; i < kNearSteps; ++i) {
      const int p = first + i * PW + lane / L;
      if (c == 0 && p < n) row[p] = out[i];
    }
  }
  __syncthreads();
  if constexpr (S::QW > 1) {
    for (int i = threadIdx.x; i < 4 / S::QW * N; i += 256) {
      const int w = i / N * S::QW, k = i % N, p = blockIdx.y * S::PAGES + i;
      float best = part[w * N + k];
#pragma unroll
      for (int j = 1; j < S::QW; ++j) best = fmaxf(best, part[(w + j) * N + k]);
      if (p < n) row[p] = best;
    }
  }
  if (threadIdx.x == 0)
    row[stride + blockIdx.y] = fmaxf(fmaxf(largest[0], largest[1]), fmaxf(largest[2], largest[3]));
}

// ------------------------------------------------------------------- choice ---
// A score as an unsigned number of the same order, a NaN above every number.
__device__ __forceinline__ uint64_t order_of(double s) {
  if (s != s) return ~0ull;
  const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0);   // -0 + 0 = 0
  return u >> 63 ? ~u : u | 1ull << 63;
}

// Where the choice of a sequence and KV head goes: the page ids in order, or the
// page words of a decode plan whose sequences are the chosen lists, each head's
// in a copy of the plan of its own. places: {first, pieces} a sequence, then for
// piece first + i the position of its first word.
struct Choice {
  int32_t* ids;
  int32_t* ordinals;
  int32_t* words;
  const int32_t* places;
  int64_t head_words, num_blocks;
  int32_t n_seqs, part_pages;
};

struct ChoiceRow {
  const Choice& c;
  const int32_t* table;
  int64_t row;
  int32_t* words;
  const int32_t* offsets;
  int pieces, width, last, tail;   // the list's last index, and its page's rows

  __device__ ChoiceRow(const Choice& ch, const int32_t* pages, int seq, int h, int n_kv_heads,
                       int columns, int chosen, int rows)
      : c(ch), table(pages), row(((int64_t)seq * n_kv_heads + h) * columns), words(nullptr),
        offsets(nullptr), pieces(1), width(columns), last(chosen - 1), tail(rows) {
    if (c.words) {
      words = c.words + h * c.head_words;
      offsets = c.places + 2 * c.n_seqs + c.places[2 * seq];
      pieces = c.places[2 * seq + 1];
    }
  }
  // the j-th chosen page is page p of the sequence
  __device__ void put(int j, int p) const { put(j, p, table[p]); }
  __device__ void put(int j, int p, int id) const {
    if ((unsigned)j >= (unsigned)width) return;   // (never: a list has `width` at most)
    c.ordinals[row + j] = p;
    if (!words) {
      c.ids[row + j] = id;
      return;
    }
    const int piece = min(j / c.part_pages, pieces - 1);
    const bool bad = id < 0 || (int64_t)id >= c.num_blocks;
    const int live = j == last ? tail : 16;
    const int64_t at = (int64_t)offsets[piece] + j - piece * c.part_pages;
    if (at < c.head_words)
      words[at] = (int)((uint32_t)(bad ? 0 : id) | ((uint32_t)(live - 1) & 15u) << 27 |
                        (bad ? 0x80000000u : 0u));
  }
  __device__ void none(int j) const {
    c.ordinals[row + j] = -1;
    if (!words) c.ids[row + j] = -1;
  }
};

// One workgroup of 256 threads a sequence and KV head. The k-th largest order
// value is found 8 bits at a time from a histogram of the values that agree
// with the bits found so far; then pages above it, and the first of those equal
// to it, are taken in page order.
__global__ __launch_bounds__(256) void select_kernel(
    const double* __restrict__ scores, int64_t stride, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, const int32_t* __restrict__ kv_lens,
    int32_t n_kv_heads, int32_t page_size, int32_t pages, int32_t width, Choice choice) {
  __shared__ int32_t hist[256], tails[256];
  __shared__ uint64_t found;
  __shared__ int32_t need;
  const int seq = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
  const int np = seq_pages(kv_indptr, kv_lens, seq, page_size, stride);
  const ChoiceRow to(choice, kv_indices + kv_indptr[seq], seq, h, n_kv_heads, width,
                     min(np, pages), kv_lens[seq] - (np - 1) * page_size);
  auto put = [&](int j, int p) { to.put(j, p); };
  if (np <= pages) {
    for (int j = tid; j < width; j += 256) {
      if (j < np) put(j, j);
      else to.none(j);
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

// The same for up to B * K pages, a page's order value in a register: B threads
// with K values each. The values of a head lie close together, so the digits
// start at the highest bit in which the largest and the smallest differ, and
// end as soon as a digit's bin holds exactly the pages still needed: two or
// three rounds, not eight.
//
// NEAR: the scores are the 32-bit sums. The cut t of those settles a page whose
// sum is more than two errors above it (in: fewer than k pages can beat it) or
// below it (out: k pages beat it). Of the pages between, the rest of the k are
// in: all of them, mostly; else their 64-bit scores decide.
constexpr int kOpenRanks = 64;   // open pages up to which each counts the others

__device__ __forceinline__ double shift_xor(double v, int m) {
  return __builtin_bit_cast(double, __shfl_xor(__builtin_bit_cast(unsigned long long, v), m));
}

template <int B, int K> struct SelectLds {
  static constexpr int W = B / 64;
  int32_t hist[256], counts[2][W * K], page[kOpenRanks], sums[2][W];
  uint64_t range[2][W], value[kOpenRanks];
  int32_t digit, above, inside;
  float q_sum[W], b_max[W];
};

template <typename U> struct Cut {
  U least;      // values from here on are taken,
  int need;     // of those equal to it (only if `ties`) the first `need`
  bool ties;
};

// The k largest of the values u[i] with bit i of `valid` (k at most their number;
// called by every thread of the workgroup).
template <typename U, int B, int K>
__device__ __forceinline__ Cut<U> find_cut(SelectLds<B, K>& l, const U* u, uint32_t valid, int k) {
  constexpr int W = B / 64, BITS = 8 * (int)sizeof(U);
  static_assert(B >= 256 && W * K <= 256, "a bin a thread, a count a lane of four");
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  U lo = ~(U)0, hi = 0;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    if (valid >> i & 1) {
      lo = u[i] < lo ? u[i] : lo;
      hi = u[i] > hi ? u[i] : hi;
    }
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const U a = (U)__shfl_xor((unsigned long long)lo, m);
    const U b = (U)__shfl_xor((unsigned long long)hi, m);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  if (lane == 0) { l.range[0][wave] = lo; l.range[1][wave] = hi; }
  if (tid < 256) l.hist[tid] = 0;
  __syncthreads();
  for (int w = 0; w < W; ++w) {
    lo = (U)l.range[0][w] < lo ? (U)l.range[0][w] : lo;
    hi = (U)l.range[1][w] > hi ? (U)l.range[1][w] : hi;
  }
  // of the values in [least, least + 2^shift) the largest `need` are in
  int shift = lo == hi ? 0 : 64 - __builtin_clzll((uint64_t)(lo ^ hi));
  Cut<U> cut{shift < BITS ? (U)(lo >> shift << shift) : (U)0, k, lo == hi};
  while (shift > 0) {
    const int next = shift > 8 ? shift - 8 : 0;
    // values that agree above `shift`, by their next bits. The largest first:
    // digit b counts in hist[255 ^ b], so that wave 0's addresses below grow with
    // the lane. Read as hist[255 - 4 l - j] they became a negative base plus an
    // offset, and those reads returned other data in every workgroup whose LDS
    // does not start at 0.
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const bool in = (valid >> i & 1) && (shift == BITS || (u[i] ^ cut.least) >> shift == 0);
      if (in) atomicAdd(&l.hist[255 ^ (int)((u[i] - cut.least) >> next)], 1);
    }
    __syncthreads();
    if (wave == 0) {
      // lane l has the bins 255 - (4 l + 0..3)
      int c[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[j] = l.hist[4 * lane + j];
        sum += c[j];
      }
      int run = sum;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_up(run, m);
        run += lane >= m ? o : 0;
      }
      int before = run - sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (before < cut.need && before + c[j] >= cut.need) {
          l.digit = 255 ^ (4 * lane + j);
          l.above = before;
          l.inside = c[j];
        }
        before += c[j];
      }
    }
    __syncthreads();
    cut.least += (U)l.digit << next;
    cut.need -= l.above;
    shift = next;
    cut.ties = l.inside > cut.need;
    if (!cut.ties) break;
    if (tid < 256) l.hist[tid] = 0;
    __syncthreads();
  }
  __syncthreads();   // l may be used again
  return cut;
}

// The sums over the workgroup of a and b.
template <int B, int K>
__device__ __forceinline__ void block_sum(SelectLds<B, K>& l, int& a, int& b) {
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    a += __shfl_xor(a, m);
    b += __shfl_xor(b, m);
  }
  if ((threadIdx.x & 63) == 0) { l.sums[0][wave] = a; l.sums[1][wave] = b; }
  __syncthreads();
  a = b = 0;
  for (int w = 0; w < B / 64; ++w) { a += l.sums[0][w]; b += l.sums[1][w]; }
}

struct NearArgs {
  const void* q; const void* lo; const void* hi;
  int64_t num_blocks;
  int32_t D, G, block_pages;     // pages of a workgroup of near_scores_kernel
};

template <typename T, bool NEAR, int B, int K>
__global__ __launch_bounds__(B) void select_rows_kernel(
    const double* __restrict__ scores, int64_t stride, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, const int32_t* __restrict__ kv_lens,
    int32_t n_kv_heads, int32_t page_size, int32_t pages, int32_t width, Choice choice,
    NearArgs na) {
  constexpr int W = B / 64;          // waves
  __shared__ SelectLds<B, K> l;
  const int seq = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63;
  // The scores go out with the lengths (a row has room for `stride` of them, and
  // what lies past the sequence's is not used).
  const double* sc = scores + ((int64_t)seq * n_kv_heads + h) * stride;
  const float* near_row = reinterpret_cast<const float*>(sc);   // scores, then maxima
  double wide_score[NEAR ? 1 : K];
  float near_score[NEAR ? K : 1];
  if (stride > pages && pages > 1) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int p = min((int64_t)i * B + tid, stride - 1);
      if constexpr (NEAR) near_score[i] = near_row[p];
      else wide_score[i] = sc[p];
    }
  }
  const int np = seq_pages(kv_indptr, kv_lens, seq, page_size, stride);
  const int32_t* table = kv_indices + kv_indptr[seq];
#pragma unroll
  for (int i = 0; i < K; ++i) {   // (here at the latest: not sunk to their first use)
    if constexpr (NEAR) asm volatile("" ::"v"(near_score[i]));
    else asm volatile("" ::"v"(wide_score[i]));
  }
  const ChoiceRow to(choice, table, seq, h, n_kv_heads, width, min(np, pages),
                     kv_lens[seq] - (np - 1) * page_size);
  if (np <= pages) {
    for (int j = tid; j < width; j += B) {
      if (j < np) to.put(j, j);
      else to.none(j);
    }
    return;
  }
  const int n = np - 1, k = pages - 1;
  if (tid == 0) to.put(k, n);
  if (k == 0) return;
  uint32_t valid = 0, sure = 0;      // bit i: page i B + tid; settled as in
  int32_t id[K];                     // (read beside the search, not after it)
#pragma unroll
  for (int i = 0; i < K; ++i) {
    valid |= (uint32_t)(i * B + tid < n) << i;
    id[i] = table[min(i * B + tid, n - 1)];
  }
  uint64_t u[K];
  Cut<uint64_t> cut;
  if constexpr (!NEAR) {
#pragma unroll
    for (int i = 0; i < K; ++i) u[i] = valid >> i & 1 ? order_of(wide_score[i]) : 0;
    cut = find_cut<uint64_t, B, K>(l, u, valid, k);
  } else {
    const T* q = (const T*)na.q + ((int64_t)seq * n_kv_heads + h) * na.G * na.D;
    // sum |q| of each query head, a head a wave; the largest bound
    float q_sum = 0.f, b_max = 0.f;
    for (int g = wave; g < na.G; g += W) {
      float t = 0.f;
      for (int d = lane; d < na.D; d += 64) t += __builtin_fabsf(Elem<T>::to_f(q[g * na.D + d]));
      t = wave_sum(t);
      q_sum = t > q_sum || t != t ? t : q_sum;
    }
    for (int i = tid; i < (n + na.block_pages - 1) / na.block_pages; i += B)
      b_max = fmaxf(b_max, near_row[stride + i]);
    b_max = wave_max(b_max);
    if (lane == 0) { l.q_sum[wave] = q_sum; l.b_max[wave] = b_max; }
    float a[K];
    uint32_t v[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
      a[i] = valid >> i & 1 ? near_score[i] : 0.f;
      const uint32_t bits = __builtin_bit_cast(uint32_t, a[i] + 0.f);
      v[i] = bits >> 31 ? ~bits : bits | 1u << 31;
    }
    const Cut<uint32_t> c32 = find_cut<uint32_t, B, K>(l, v, valid, k);   // (a barrier inside)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      q_sum = l.q_sum[w] > q_sum || l.q_sum[w] != l.q_sum[w] ? l.q_sum[w] : q_sum;
      b_max = fmaxf(b_max, l.b_max[w]);
    }
    const float t = __builtin_bit_cast(
        float, c32.least >> 31 ? c32.least ^ 1u << 31 : ~c32.least);
    const float e = 2.01f * near(q_sum, b_max, na.D) + 4.8e-7f * __builtin_fabsf(t);
    uint32_t open = 0;
    int n_sure = 0, n_open = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      if (!(valid >> i & 1)) continue;
      // (a comparison with something that is no number settles nothing)
      const float d = a[i] - t;
      if (e < INFINITY && d > e) { sure |= 1u << i; ++n_sure; }
      else if (!(e < INFINITY && d < -e)) { open |= 1u << i; ++n_open; }
    }
    block_sum(l, n_sure, n_open);
    // (all k may be settled with pages open below them: t can lie between the
    // k-th sum and the next)
    if (n_sure == k || n_open == k - n_sure) {
      if (n_sure < k) sure |= open;
      valid = 0;
      cut = Cut<uint64_t>{0, 0, false};
    } else {
      // 64-bit scores of the open pages, one of a wave at a time: D / 8 lanes a
      // query head, 64 / (D / 8) heads side by side
      typedef T vec __attribute__((ext_vector_type(8)));
      const int L = na.D / 8, side = 64 / L, c = lane % L;
#pragma unroll
      for (int i = 0; i < K; ++i) {
        u[i] = 0;
        for (uint64_t who = __builtin_amdgcn_ballot_w64(open >> i & 1); who; who &= who - 1) {
          const int owner = __builtin_ctzll(who);
          int64_t id = table[i * B + wave * 64 + owner];
          if (id < 0 || id >= na.num_blocks) id = 0;      // (flagged by the first pass)
          const int64_t off = (id * n_kv_heads + h) * na.D + c * 8;
          const vec x = *reinterpret_cast<const vec*>((const T*)na.lo + off);
          const vec y = *reinterpret_cast<const vec*>((const T*)na.hi + off);
          double best = -INFINITY;
          for (int g0 = 0; g0 < na.G; g0 += side) {
            const vec z = *reinterpret_cast<const vec*>(
                q + min(g0 + lane / L, na.G - 1) * na.D + c * 8);
            double s = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float f = Elem<T>::to_f(z[j]);
              s = __builtin_fma((double)f, (double)Elem<T>::to_f(f < 0.f ? x[j] : y[j]), s);
            }
            for (int m = 1; m < L; m <<= 1) s += shift_xor(s, m);
            for (int m = L; m < 64; m <<= 1) {
              const double o = shift_xor(s, m);
              s = o != o || o > s ? o : s;
            }
            best = s != s || s > best ? s : best;
          }
          if (lane == owner) u[i] = order_of(best);
        }
      }
      valid = open;
      if (n_open <= kOpenRanks) {
        // few: each counts those that beat it
        if (tid == 0) l.digit = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < K; ++i) {
          if (open >> i & 1) {
            const int at = atomicAdd(&l.digit, 1);
            l.value[at] = u[i];
            l.page[at] = i * B + tid;
          }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < K; ++i) {
          if (open >> i & 1) {
            int beaten = 0;
            for (int e = 0; e < n_open; ++e)
              beaten += l.value[e] > u[i] || (l.value[e] == u[i] && l.page[e] < i * B + tid);
            if (beaten < k - n_sure) sure |= 1u << i;
          }
        }
        valid = 0;
        cut = Cut<uint64_t>{0, 0, false};
      } else {
        cut = find_cut<uint64_t, B, K>(l, u, valid, k - n_sure);
      }
    }
  }
  // Page order is (i, thread): a count a wave and i, and their sums before each.
  uint32_t in = sure, eq = 0;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    if (valid >> i & 1) {
      in |= (uint32_t)(u[i] >= cut.least) << i;
      eq |= (uint32_t)(cut.ties && u[i] == cut.least) << i;
    }
    const uint64_t bi = __builtin_amdgcn_ballot_w64(in >> i & 1);
    const uint64_t be = __builtin_amdgcn_ballot_w64(eq >> i & 1);
    if (lane == 0) {
      l.counts[0][i * W + wave] = __builtin_popcountll(bi & ~be);
      l.counts[1][i * W + wave] = __builtin_popcountll(be);
    }
  }
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      constexpr int C = (W * K + 63) / 64;
      int c[C], sum = 0;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        c[j] = lane * C + j < W * K ? l.counts[t][lane * C + j] : 0;
        sum += c[j];
      }
      int run = sum;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_up(run, m);
        run += lane >= m ? o : 0;
      }
      run -= sum;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if (lane * C + j < W * K) l.counts[t][lane * C + j] = run;
        run += c[j];
      }
    }
  }
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const uint64_t bi = __builtin_amdgcn_ballot_w64(in >> i & 1);
    const uint64_t be = __builtin_amdgcn_ballot_w64(eq >> i & 1);
    const int before = l.counts[0][i * W + wave] + __builtin_popcountll(bi & ~be & below);
    const int e = l.counts[1][i * W + wave] + __builtin_popcountll(be & below);
    if ((in >> i & 1) && (!(eq >> i & 1) || e < cut.need))
      to.put(before + (cut.ties ? min(e, cut.need) : 0), i * B + tid, id[i]);
  }
}

struct ScoreArgs {
  const void* q; const void* lo; const void* hi; int64_t nb;
  const int32_t* indptr; const int32_t* indices; const int32_t* kv_lens;
  int32_t n_seqs, Hkv, page_size, pages, max_pages; double* scores; int32_t* status;
};
constexpr int kSelectMax = 1024 * 16;   // pages select_rows_kernel holds
// Elements of lo (over KV heads and sequences, were every list as long as the
// longest) from which the scores run in 32 bits first: the choice then takes 4 to 5 us more, for the pages left
// open. us of scores and choice, 32 bits against 64: 1M elements 16.6 and 14.6,
// 3M 17.5 and 15.9, 25M 27.7 and 29.0, 61M 45.4 and 54.2.
constexpr int64_t kNearLeast = 16 << 20;
typedef void (*ScoreFn)(const ScoreArgs&, hipStream_t);

template <typename T, int D, int G>
static void launch_scores(const ScoreArgs& a, hipStream_t s) {
  constexpr int PAGES = ScoreShape<T, D, G>::PAGES;
  hipLaunchKernelGGL((score_rows_kernel<T, D, G>),
                     dim3((unsigned)a.Hkv, (unsigned)((a.max_pages - 1 + PAGES - 1) / PAGES),
                          (unsigned)a.n_seqs),
                     dim3(256), 0, s, (const T*)a.q, (const T*)a.lo, (const T*)a.hi, a.nb, a.indptr,
                     a.indices, a.kv_lens, a.Hkv, a.page_size, a.pages, (int64_t)a.max_pages,
                     a.scores, a.status);
}

template <typename T, int D, int G>
static void launch_near(const ScoreArgs& a, hipStream_t s) {
  constexpr int PAGES = NearShape<T, D, G>::PAGES;
  hipLaunchKernelGGL((near_scores_kernel<T, D, G>),
                     dim3((unsigned)a.Hkv, (unsigned)((a.max_pages - 1 + PAGES - 1) / PAGES),
                          (unsigned)a.n_seqs),
                     dim3(256), 0, s, (const T*)a.q, (const T*)a.lo, (const T*)a.hi, a.nb, a.indptr,
                     a.indices, a.kv_lens, a.Hkv, a.page_size, a.pages, (int64_t)a.max_pages,
                     (float*)a.scores, a.status);
}

// The 32-bit scores of a 16-bit pool, and the pages of its workgroups.
struct NearFn { ScoreFn launch; int block_pages; };

template <typename T, int D>
static NearFn near_g(int G) {
  switch (G) {
    case 1: return {launch_near<T, D, 1>, NearShape<T, D, 1>::PAGES};
    case 2: return {launch_near<T, D, 2>, NearShape<T, D, 2>::PAGES};
    case 4: return {launch_near<T, D, 4>, NearShape<T, D, 4>::PAGES};
    case 8: return {launch_near<T, D, 8>, NearShape<T, D, 8>::PAGES};
    case 16: return {launch_near<T, D, 16>, NearShape<T, D, 16>::PAGES};
    default: return {nullptr, 0};
  }
}

template <typename T, int D>
static ScoreFn score_g(int G) {
  switch (G) {
    case 1: return launch_scores<T, D, 1>;
    case 2: return launch_scores<T, D, 2>;
    case 4: return launch_scores<T, D, 4>;
    case 8: return launch_scores<T, D, 8>;
    case 16: return launch_scores<T, D, 16>;
    default: return nullptr;
  }
}

template <typename T>
static ScoreFn score_fn(int32_t D, int32_t G) {
  return D == 64 ? score_g<T, 64>(G) : D == 128 ? score_g<T, 128>(G) : nullptr;
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
  auto pick = [&](auto type) {
    typedef decltype(type) T;
    constexpr int W = 16 / (int)sizeof(T);
    if (V == 1) go(page_bounds_kernel<T, 1, 0>);
    else if (page_size == 16) go(page_bounds_kernel<T, W, 16>);
    else go(page_bounds_kernel<T, W, 0>);
  };
  if (dtype == PKV_DTYPE_F16) pick(_Float16{});
  else if (dtype == PKV_DTYPE_BF16) pick(__bf16{});
  else pick(float{});
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

extern "C" int pkv_select_pages(const void* q, const void* lo, const void* hi, int64_t num_blocks,
                                const int32_t* kv_indptr, const int32_t* kv_indices,
                                const int32_t* kv_lens, int32_t n_seqs, int32_t max_pages,
                                int32_t pages, int32_t n_heads, int32_t n_kv_heads,
                                int32_t head_dim, int32_t page_size, int32_t dtype,
                                double* scores, int32_t* ids, int32_t* ordinals,
                                int32_t* words, const int32_t* places, int64_t head_words,
                                int32_t part_pages, int32_t* status_word, void* stream) {
  int rc = check_geometry(n_heads, n_kv_heads, head_dim, page_size, dtype);
  if (rc) return rc;
  if (n_seqs < 0 || n_seqs > 65535 || n_kv_heads > 65535 || max_pages <= 0 || pages <= 0)
    return fail(PKV_ERR_INVALID, "max_pages and pages must be positive, and one call takes up to "
                "65535 sequences and KV heads");
  if (n_seqs == 0) return PKV_OK;
  if (!q || !lo || !hi || !kv_indptr || !kv_indices || !kv_lens || !ordinals ||
      (max_pages > pages && !scores) || (words ? !places : !ids))
    return fail(PKV_ERR_INVALID, "null pointer argument");
  if (words && (part_pages < 1 || head_words < 1 || page_size != 16 ||
                num_blocks > (1LL << 27)))
    return fail(PKV_ERR_INVALID, "page words need a plan (pkv_plan_selected)");
  const int32_t width = std::min(pages, max_pages);
  hipStream_t s = (hipStream_t)stream;
  NearFn near{nullptr, 0};
  if (max_pages > pages && pages > 1) {
    const uintptr_t at = (uintptr_t)q | (uintptr_t)lo | (uintptr_t)hi |
                         (uintptr_t)((int64_t)head_dim * elem_bytes(dtype));
    const ScoreArgs args{q, lo, hi, num_blocks, kv_indptr, kv_indices, kv_lens, n_seqs, n_kv_heads,
                         page_size, pages, max_pages, scores, status_word};
    const bool wide = at % 16 == 0;
    const int32_t G = n_heads / n_kv_heads;
    auto score = [&](auto type) {
      typedef decltype(type) T;
      if constexpr (sizeof(T) == 2) {
        // (a list that fits the registers of select_rows_kernel)
        if (wide && max_pages <= kSelectMax &&
            (int64_t)n_seqs * n_kv_heads * max_pages * head_dim >= kNearLeast)
          near = head_dim == 64 ? near_g<T, 64>(G) : head_dim == 128 ? near_g<T, 128>(G) : near;
        if (near.launch) return near.launch(args, s);
      }
      // (a grid of up to 65535 workgroups of at least 8 pages)
      const ScoreFn fn = wide && max_pages <= 8 * 65535 ? score_fn<T>(head_dim, G) : nullptr;
      if (fn) return fn(args, s);
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((max_pages + 62) / 64), (unsigned)n_kv_heads,
                                        (unsigned)n_seqs),
                           dim3(64), 0, s, (const T*)q, (const T*)lo, (const T*)hi, num_blocks,
                           kv_indptr, kv_indices, kv_lens, n_heads, n_kv_heads, head_dim,
                           page_size, pages, (int64_t)max_pages, scores, status_word);
      };
      if (wide) go(score_kernel<T, 16 / (int)sizeof(T)>);
      else go(score_kernel<T, 1>);
    };
    if (dtype == PKV_DTYPE_F16) score(_Float16{});
    else if (dtype == PKV_DTYPE_BF16) score(__bf16{});
    else score(float{});
    PKV_LAUNCH_CHECK();
  }
  const Choice choice{ids, ordinals, words, places, head_words, num_blocks, n_seqs, part_pages};
  const NearArgs na{q, lo, hi, num_blocks, head_dim, n_heads / n_kv_heads, near.block_pages};
  auto choose = [&](auto kernel, int threads, auto... more) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)n_kv_heads, (unsigned)n_seqs), dim3(threads), 0, s,
                       scores, (int64_t)max_pages, kv_indptr, kv_indices, kv_lens, n_kv_heads,
                       page_size, pages, width, choice, more...);
  };
  auto rows = [&](auto type, auto is_near) {
    typedef decltype(type) T;
    constexpr bool N = decltype(is_near)::value;
    if (max_pages <= 256 * 4) choose(select_rows_kernel<T, N, 256, 4>, 256, na);
    else if (max_pages <= 1024 * 4) choose(select_rows_kernel<T, N, 1024, 4>, 1024, na);
    else choose(select_rows_kernel<T, N, 1024, 16>, 1024, na);
  };
  if (max_pages > kSelectMax) choose(select_kernel, 256);
  else if (!near.launch) rows(float{}, std::false_type{});
  else if (dtype == PKV_DTYPE_F16) rows(_Float16{}, std::true_type{});
  else rows(__bf16{}, std::true_type{});
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}
