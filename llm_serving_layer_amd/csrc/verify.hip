// Verification of drafted tokens against the target's logits, from given uniform
// numbers. A sequence of n rows (the last accepted token, then n - 1 drafts) keeps
// the drafts x_j for which u_j q_j(x_j) < p_j(x_j), up to the first that does not
// stand; p_j is the softmax of row j's logits over the temperature, q_j the
// drafting distribution (1 at x_j where none is given). The token behind them is
// drawn from max(p - q, 0) where a draft fell (p where that is nothing), from p
// behind a run that stands whole: the first whose running sum of weights exceeds
// u_last times the weights' sum. Weights below 2^-1000 of a row's largest count as
// nothing. At a temperature of 0 or below a draft stands if it is the row's
// greedy pick, which is the token otherwise.
//
// These are decisions, and are made as in 64 bits; what can be done in 32 is.
//  * verify_stats_kernel reads every row once (the operator's bound: HBM), a row
//    over several workgroups: maximum, its first place, and the sum of 2^((l -
//    max) c), c = log2 e / temperature, in 32 bits.
//  * verify_draw_kernel: each workgroup of a sequence repeats its tests on those
//    statistics (a few loads; no launch of its own). A test closer than the sum's
//    error takes the row's sum in 64 bits. The workgroups then sum their units of
//    the one row that a token is drawn from in 64 bits: an exponential is a table
//    of 256 entries in LDS and a polynomial of degree 4, some 20 instructions, on
//    n rows instead of all. The last one to arrive finds the token, except where
//    the row's whole sum is needed first:
//  * verify_rest_kernel, with draft probabilities: the same over max(p - q, 0).
//    In 32 bits the sum's error would move the border of every token behind it.
// 64 sequences of 2 to 6 rows of 128256 bf16 logits, fp32 draft probabilities: 17.4 (64
// MB, 3.7 TB/s) + 18.1 + 18.3 us; 24 of 9 rows in fp32 21.2 (5.2 TB/s) + 14.4 + 14.4; one
// sequence of 5 rows 4.5 + 5.8 + 8.8, a chain of waits. Of the second and third kernel's 18
// us, vector instructions are 6 and 4: the rest is each workgroup's table and decision
// before its first useful load, the arrival, and the last one's search, not timed apart.
#include <algorithm>

#include "mfma.h"

namespace pkv {

constexpr int kVT = 256;            // threads of a workgroup
constexpr int kMaxSplits = 64;      // of a row: a lane each
constexpr int kChunks = 8;          // of 16 bytes a thread and round, in the first kernel
                                    // (249 rows of 128256 in bf16: 17.4 us; 4 take 1.2 more)

struct RowStats { float m, z; int32_t arg, pad; };

// A sequence's decision: how many drafts stand, and the row that follows.
struct Decision {
  int32_t run, row, token;   // token: taken as it is, or -1: drawn from the row
  int32_t banned;            // the draft that fell, without draft probabilities; -1
  int32_t rest, pad;         // drawn from max(p - q, 0)
  double m, c;               // the row's largest logit, log2 e / temperature
};

struct Verify {
  const void* logits;
  const void* probs;
  const int64_t* tokens;
  const int32_t *cu, *owner;
  const float *numbers, *temps;
  RowStats* stats;
  Decision* decisions;
  double *sums, *rest;              // of a sequence's units: 2^x, max(2^x - q z, 0)
  int32_t* counters;                // two a sequence; cleared by the first kernel
  int64_t *ids, *accepted;
  int64_t row_stride, probs_stride, width;
  int32_t n_rows, n_seqs, vocab, splits, parts, units, cells;
  float temp, error;                // error: of a row's 32-bit sum, relative
};

// The part s of n of a row: elements [begin, end), the inner borders on 16-byte
// boundaries of the row's memory.
template <typename T>
__device__ __forceinline__ void part_of(const T* row, int vocab, int s, int n, int& begin, int& end) {
  constexpr int E = 16 / (int)sizeof(T);
  const int head = min((int)((-(uintptr_t)row & 15) / sizeof(T)), vocab);
  const int chunks = (vocab - head) / E, per = (chunks + n - 1) / n;
  begin = s == 0 ? 0 : head + min(s * per, chunks) * E;
  end = s == n - 1 ? vocab : head + min((s + 1) * per, chunks) * E;
}

// What a temperature divides by: 1 for greedy rows; at most the largest finite float,
// so that log2 e / temperature is not 0, and a logit of -inf keeps no weight.
__device__ __forceinline__ float divisor(float t) { return t > 0.f ? fminf(t, 0x1.fffffep127f) : 1.f; }

template <typename T>
__global__ __launch_bounds__(kVT) void verify_stats_kernel(Verify a) {
  constexpr int E = 16 / (int)sizeof(T), U = kChunks;
  typedef T TV __attribute__((ext_vector_type(E)));
  const int r = blockIdx.x / a.splits, s = blockIdx.x - r * a.splits;
  const int tid = threadIdx.x;
  if (s == 0 && r < a.n_seqs && tid < 2) a.counters[2 * r + tid] = 0;
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  int begin, end;
  part_of(row, a.vocab, s, a.splits, begin, end);
  const int seq = a.owner[r];
  const float t = a.temps ? (seq >= 0 && seq < a.n_seqs ? a.temps[seq] : 1.f) : a.temp;
  const float c = fminf(kLog2e / divisor(t), 0x1p100f);
  float m = -INFINITY, z = 0.f;
  int arg = 0x7fffffff;             // the thread's first place of m, or its chunk's start
  auto scalar = [&](int i) {
    const float l = Elem<T>::to_f(row[i]);
    const float mn = fmaxf(m, l);
    if (l > m || arg == 0x7fffffff) arg = i;
    const float ref = mn == -INFINITY ? 0.f : mn;
    z = z * __builtin_amdgcn_exp2f((m - ref) * c) + __builtin_amdgcn_exp2f((l - ref) * c);
    m = mn;
  };
  const int head = s == 0 ? min((int)((-(uintptr_t)row & 15) / sizeof(T)), end) : 0;
  const int body = begin + head, chunks = (end - body) / E;
  if (tid < head) scalar(tid);
  for (int c0 = 0; c0 < chunks; c0 += U * kVT) {
    TV w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = c0 + u * kVT + tid;
      if (k < chunks)
        w[u] = __builtin_nontemporal_load(reinterpret_cast<const TV*>(row + body + (int64_t)k * E));
      else
#pragma unroll
        for (int e = 0; e < E; ++e) w[u][e] = (T)-INFINITY;
    }
    float top = m;
    const int live = min(U, (chunks - c0 + kVT - 1) / kVT);   // of the U, uniform
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= live) break;
      TV x = w[u];
      float cm = Elem<T>::to_f(x[0]);
#pragma unroll
      for (int e = 1; e < E; ++e) cm = fmaxf(cm, Elem<T>::to_f(x[e]));
      const int k = c0 + u * kVT + tid;
      const bool gt = k < chunks && (cm > top || arg == 0x7fffffff);
      arg = gt ? body + k * E : arg;
      top = fmaxf(top, cm);
    }
    const float ref = top == -INFINITY ? 0.f : top, rc = -ref * c;
    z *= __builtin_amdgcn_exp2f((m - ref) * c);
    m = top;
    if (__builtin_fabsf(rc) < 0x1p80f) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u >= live) break;
#pragma unroll
        for (int e = 0; e < E; ++e)
          z += __builtin_amdgcn_exp2f(__builtin_fmaf(Elem<T>::to_f(w[u][e]), c, rc));
      }
    } else {                         // (far from 1: the products may overflow)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u >= live) break;
#pragma unroll
        for (int e = 0; e < E; ++e)
          z += __builtin_amdgcn_exp2f((Elem<T>::to_f(w[u][e]) - ref) * c);
      }
    }
  }
  const int tail = body + chunks * E;
  if (tail + tid < end) scalar(tail + tid);
  // the threads meet: the largest, its first place, the sum. (Places are those of
  // chunks: equal maxima in one chunk are told apart at the end.)
  __shared__ float sm[kVT / 64], sz[kVT / 64];
  __shared__ int sa[kVT / 64];
  const float wm = wave_max(m), ref = wm == -INFINITY ? 0.f : wm;
  z = wave_sum(z * __builtin_amdgcn_exp2f((m - ref) * c));
  int first = m == wm ? arg : 0x7fffffff;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) first = min(first, __shfl_xor(first, off, 64));
  if ((tid & 63) == 0) {
    sm[tid >> 6] = wm;
    sz[tid >> 6] = z;
    sa[tid >> 6] = first;
  }
  __syncthreads();
  if (tid) return;
  float bm = -INFINITY, bz = 0.f;
  int ba = 0x7fffffff;
#pragma unroll
  for (int w = 0; w < kVT / 64; ++w) bm = fmaxf(bm, sm[w]);
  const float br = bm == -INFINITY ? 0.f : bm;
#pragma unroll
  for (int w = 0; w < kVT / 64; ++w) {
    bz += sz[w] * __builtin_amdgcn_exp2f((sm[w] - br) * c);
    if (sm[w] == bm) ba = min(ba, sa[w]);
  }
  if (ba < end) {
    if (ba >= body && ba < tail) {   // (a chunk's start, read again in one load)
      const TV w = *reinterpret_cast<const TV*>(row + ba);
      int place = 0;
#pragma unroll
      for (int e = E - 1; e > 0; --e) place = Elem<T>::to_f(w[e]) == bm ? e : place;
      ba += Elem<T>::to_f(w[0]) == bm ? 0 : place;
    }
  } else {
    ba = begin;                      // (nothing but NaN, or an empty part)
  }
  a.stats[(int64_t)r * a.splits + s] = RowStats{bm, bz, ba, 0};
}

// ------------------------------------------------------------ 64-bit sums ---

// 2^(j / 256)
__device__ __forceinline__ void fill_table(double* table) {
  for (int j = threadIdx.x; j < 256; j += blockDim.x) table[j] = exp2((double)j / 256.0);
  __syncthreads();
}
// 2^x for x <= 0, 0 below -1000 (and for NaN): x = n / 256 + g, |g| <= 2^-9; 2^g =
// e^(g ln 2) by its series, the rest below 2^-54.
__device__ __forceinline__ double exp2_64(double x, const double* table) {
  constexpr double kMagic = 6755399441055744.0 / 256.0;   // 1.5 2^52 / 256: adds round to n / 256
  constexpr double kLn2 = 0.693147180559945309417;
  const double at = x + kMagic;
  const double g = x - (at - kMagic);
  const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, at);
  double p = __builtin_fma(g, kLn2 * kLn2 * kLn2 * kLn2 / 24.0, kLn2 * kLn2 * kLn2 / 6.0);
  p = __builtin_fma(g, p, kLn2 * kLn2 / 2.0);
  p = __builtin_fma(g, p, kLn2);
  const double base = table[n & 255];
  const double y = __builtin_fma(base * g, p, base);
  const uint64_t bits = __builtin_bit_cast(uint64_t, y) + ((uint64_t)(uint32_t)(n >> 8) << 52);
  return x >= -1000.0 ? __builtin_bit_cast(double, bits) : 0.0;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// v plus the lower lanes' values
__device__ __forceinline__ double wave_scan64(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double o = __shfl_up(v, off, 64);
    v += lane >= off ? o : 0.0;
  }
  return v;
}
// The drawing kernels' cells: eight elements of a row, a thread's step. (These
// kernels run their code once or twice, so its length counts as well, by the
// instruction cache's misses: their loops are rolled.)
constexpr int kDT = 512, kCell = 8, kPart = kDT * kCell;

// Eight values from wherever they lie, read where they are used.
template <typename Q> struct Eight {
  typedef Q QV __attribute__((ext_vector_type(8)));
  struct __attribute__((packed, aligned(sizeof(Q)))) Loose { QV v; };
  QV v;
  __device__ __forceinline__ void load(const Q* row, int i, int n) {
    if (i + 8 <= n) {
      v = reinterpret_cast<const Loose*>(row + i)->v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = row[min(i + e, n - 1)];
    }
  }
};

struct DrawLds {
  double table[256];
  double sums[kMaxSplits][kDT / 64], waves[kDT / 64];   // of units by wave
  RowStats rows[64];
  int flags[64];
  int last, found;
};

// The sum over the workgroup, in every thread.
__device__ __forceinline__ double block_sum64(double v, double* lds) {
  v = wave_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kDT / 64; ++w) s += lds[w];
  return s;
}

// The weights 2^((l - m) c), or, with probabilities p, max(2^((l - m) c) iz - p, 0),
// of cells; none at `banned` and past the vocabulary.
struct Weigh {
  const double* table;
  double m, c, iz;
  int banned, vocab;
  template <typename T, typename Q>
  __device__ __forceinline__ double operator()(const Eight<T>& l, const Eight<Q>& p, bool rest, int i,
                                               double (&w)[kCell]) const {
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < kCell; ++e) {
      double x = exp2_64(((double)Elem<T>::to_f(l.v[e]) - m) * c, table);
      if (rest) {
        x = x * iz - (double)Elem<Q>::to_f(p.v[e]);
        x = x > 0.0 ? x : 0.0;
      }
      w[e] = x;
    }
    if (i + kCell > vocab || (unsigned)(banned - i) < (unsigned)kCell) {
#pragma unroll
      for (int e = 0; e < kCell; ++e)
        if (i + e >= vocab || i + e == banned) w[e] = 0.0;
    }
#pragma unroll
    for (int e = 0; e < kCell; ++e) sum += w[e];
    return sum;
  }
};

// The sum of a thread's cells, from element `at` on, `step` elements apart, `count`
// of them; the next one is on its way while one is weighed. w: the last one's.
template <typename T, typename Q>
__device__ __forceinline__ double weigh_run(const T* row, const Q* q, int at, int step, int count,
                                            const Weigh& weigh, double (&w)[kCell]) {
  Eight<T> l, l2;
  Eight<Q> p{}, p2{};
  const int n = weigh.vocab, last = n - 1;
  l.load(row, min(at, last), n);
  if (q) p.load(q, min(at, last), n);
  double sum = 0.0;
#pragma unroll 1
  for (int r = 0; r < count; ++r, at += step) {
    const int next = min(r + 1 < count ? at + step : at, last);
    l2.load(row, next, n);
    if (q) p2.load(q, next, n);
    sum += weigh(l, p, q != nullptr, at, w);
    l = l2;
    p = p2;
  }
  return sum;
}

// The sums of units [u0, u1) by wave, into lds: `cells` of a thread's a unit, the next
// one on its way while one is weighed.
template <typename T, typename Q>
__device__ __forceinline__ void weigh_units(const T* row, const Q* q, int u0, int u1, int cells,
                                            const Weigh& weigh, double (&lds)[kMaxSplits][kDT / 64]) {
  const int n = weigh.vocab, last = n - 1, tid = threadIdx.x;
  Eight<T> l, l2;
  Eight<Q> p{}, p2{};
  int at = (u0 * kDT + tid) * cells * kCell;
  l.load(row, min(at, last), n);
  if (q) p.load(q, min(at, last), n);
  double sum = 0.0;
  int u = 0;
#pragma unroll 1
  for (int j = 1; u < u1 - u0; ++j) {
    const int next = at + (j < cells ? 1 : (kDT - 1) * cells + 1) * kCell;
    l2.load(row, min(next, last), n);
    if (q) p2.load(q, min(next, last), n);
    double w[kCell];
    sum += weigh(l, p, q != nullptr, at, w);
    at = next;
    l = l2;
    p = p2;
    if (j < cells) continue;
    sum = wave_sum64(sum);
    if ((tid & 63) == 0) lds[u][tid >> 6] = sum;
    sum = 0.0;
    j = 0;
    ++u;
  }
}

// Decides a sequence (uniform over the workgroup).
template <typename T, typename Q>
__device__ Decision decide(const Verify& a, int seq, DrawLds& lds) {
  const int r0 = a.cu[seq], n = a.cu[seq + 1] - r0;
  const float t = a.temps ? a.temps[seq] : a.temp;
  const bool greedy = !(t > 0.f);
  const double c = 1.44269504088896340736 / (double)divisor(t);
  const float cf = fminf((float)c, 0x1p100f);
  const T* logits = reinterpret_cast<const T*>(a.logits);
  const int tid = threadIdx.x, lane = tid & 63;
  Decision d;
  d.c = c;
  d.run = n - 1;
  RowStats b{};
  // 64 rows at a time: a thread a row reads what its test needs, a wave a row its
  // statistics, a lane a part (there are at most 64); then the threads test.
  for (int j0 = 0; j0 < n; j0 += 64) {
    const int m = min(64, n - j0);
    int64_t x = -1;
    float u = 0.f, lx = 0.f, qx = 1.f;
    if (tid < m && j0 + tid < n - 1) {
      const int r = r0 + j0 + tid;
      x = a.tokens[r + 1];
      u = a.numbers[r];
      if (x >= 0 && x < a.vocab) {
        lx = Elem<T>::to_f(logits[r * a.row_stride + x]);
        if (a.probs)
          qx = Elem<Q>::to_f(
              reinterpret_cast<const Q*>(a.probs)[(int64_t)(r - seq) * a.probs_stride + x]);
      } else {
        x = -1;
      }
    }
    for (int j = tid >> 6; j < m; j += kDT / 64) {
      const RowStats st = lane < a.splits ? a.stats[(int64_t)(r0 + j0 + j) * a.splits + lane]
                                          : RowStats{-INFINITY, 0.f, 0x7fffffff, 0};
      const float top = wave_max(st.m), ref = top == -INFINITY ? 0.f : top;
      const float z = wave_sum(st.z * __builtin_amdgcn_exp2f((st.m - ref) * cf));
      int arg = st.m == top ? st.arg : 0x7fffffff;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) arg = min(arg, __shfl_xor(arg, off, 64));
      if (lane == 0) lds.rows[j] = RowStats{top, z, arg, 0};
    }
    __syncthreads();
    double ex = 0.0, need = 0.0;
    if (tid < m) {
      const RowStats s = lds.rows[tid];
      int state = 0;                 // 0: falls, 1: stands, 2: too close to tell
      if (x >= 0 && s.z == s.z && s.m != -INFINITY) {   // (else: no distribution)
        if (greedy) {
          state = s.arg == x;
        } else {
          ex = exp2_64(((double)lx - (double)s.m) * c, lds.table);
          need = (double)u * (double)qx;
          const double sum = need * (double)s.z;
          // the sum's error, relative: its terms' and their sums' (a.error), and what
          // the rounding of m c does to every exponent; none is known where c was cut
          // to 2^100, or is so small that l - m may overflow and still have weight
          const double error =
              c < 0x1p100 && c > 0x1p-120
                  ? (double)a.error + fmin(fabs((double)s.m * c), 0x1p80) * 0x1p-23
                  : INFINITY;
          state = fabs(sum - ex) <= error * fabs(sum) ? 2 : sum < ex;
        }
      }
      lds.flags[tid] = state;
    }
    __syncthreads();
    int at = -1;                     // the run's end in these rows
    for (int i = 0; i < m; ++i) {
      const int s = lds.flags[i];
      if (s == 1) continue;
      if (s == 2) {                  // the row's sum in 64 bits
        const double top = (double)lds.rows[i].m;
        double w[kCell];
        const double z = block_sum64(
            weigh_run(logits + (r0 + j0 + i) * a.row_stride, (const Q*)nullptr, tid * kCell, kPart,
                      (a.vocab + kPart - 1) / kPart, Weigh{lds.table, top, c, 1.0, -1, a.vocab}, w),
            lds.waves);
        if (tid == i) lds.last = need < ex / z;
        __syncthreads();
        const bool stands = lds.last;
        __syncthreads();
        if (stands) continue;
      }
      at = i;
      break;
    }
    if (at >= 0) {
      d.run = j0 + at;
      b = lds.rows[at];
    }
    __syncthreads();                 // rows and flags are free again
    if (at >= 0) break;
  }
  d.row = r0 + d.run;
  d.m = b.m;
  d.token = -1;
  const bool none = !(b.z == b.z) || b.m == -INFINITY;   // no distribution
  if (greedy || none) d.token = b.arg;
  if (!(b.z == b.z)) {               // a NaN, or +inf: torch's order, the first NaN first
    if (tid == 0) lds.found = 0x7fffffff;
    __syncthreads();
    for (int i = tid; i < a.vocab; i += kDT) {
      const float l = Elem<T>::to_f(logits[d.row * a.row_stride + i]);
      if (l != l) atomicMin(&lds.found, i);
    }
    __syncthreads();
    if (lds.found != 0x7fffffff) d.token = lds.found;
    __syncthreads();
  }
  d.rest = d.run < n - 1 && a.probs;
  d.banned = -1;
  if (d.run < n - 1 && !a.probs) {
    const int64_t x = a.tokens[d.row + 1];
    if (x >= 0 && x < a.vocab) d.banned = (int)x;
  }
  return d;
}

// Sums the units of part s of the row that a sequence draws from; the workgroup that is
// the last to (counter k) finds the token: the unit whose running sum passes the
// target, in it the thread, its element. Returns it there (-1: no weight at all), -2
// in the others. sums: the units', beyond the XCDs' caches.
enum DrawMode { kSumOnly, kCounted, kKnown };   // kKnown: sums hold all units' already

template <typename T, typename Q>
__device__ int draw(const Verify& a, int seq, int s, const Decision& d, const T* row, const Q* q,
                    double iz, int k, double* sums, DrawMode mode, DrawLds& lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, per = a.cells;
  const Weigh weigh{lds.table, d.m, d.c, iz, d.banned, a.vocab};
  if (mode != kKnown) {
    const int u0 = s * a.units / a.parts, u1 = (s + 1) * a.units / a.parts;
    weigh_units(row, q, u0, u1, per, weigh, lds.sums);
    __syncthreads();
    if (wave == 0) {
      double sum = 0.0;
      if (tid < u1 - u0)
#pragma unroll
        for (int w = 0; w < kDT / 64; ++w) sum += lds.sums[tid][w];
      if (mode == kSumOnly) {
        if (tid < u1 - u0) sums[u0 + tid] = sum;
      } else {
        if (tid < u1 - u0)
          __hip_atomic_store(sums + u0 + tid, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (tid == 0)
          lds.last = __hip_atomic_fetch_add(a.counters + 2 * seq + k, 1, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT) == a.parts - 1;
      }
    }
    if (mode == kSumOnly) return -2;
    __syncthreads();
    if (!lds.last) return -2;
  }
  // (every wave the same: a lane a unit)
  const double own =
      lane < a.units ? __hip_atomic_load(sums + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                     : 0.0;
  const double upto = wave_scan64(own);
  const double target = (double)a.numbers[a.cu[seq + 1] - 1] * __shfl(upto, 63, 64);
  const uint64_t passed = __builtin_amdgcn_ballot_w64(own > 0.0 && upto > target);
  const uint64_t some = __builtin_amdgcn_ballot_w64(own > 0.0);
  if (!some) return -1;
  // (a number of 1, or the last sum's rounding: the last weight of all)
  const bool past = passed;
  const int unit = past ? __builtin_ctzll(passed) : 63 - __builtin_clzll(some);
  const double base = past ? __shfl(upto - own, unit, 64) : 0.0;
  {
    const int first = (unit * kDT + tid) * per * kCell;
    const int count = first < a.vocab ? min(per, (a.vocab - first + kCell - 1) / kCell) : 0;
    double w[kCell] = {};
    const double mine = weigh_run(row, q, first, kCell, count, weigh, w);
    const double scan = wave_scan64(mine);
    __syncthreads();
    if (lane == 63) lds.waves[wave] = scan;
    __syncthreads();
    double run = base + (scan - mine);
    for (int v = 0; v < wave; ++v) run += lds.waves[v];
    const uint64_t over = __builtin_amdgcn_ballot_w64(past && mine > 0.0 && run + mine > target);
    const uint64_t any = __builtin_amdgcn_ballot_w64(mine > 0.0);
    if (lane == 0) {
      lds.flags[wave] = over ? tid + __builtin_ctzll(over) : -1;
      lds.flags[kDT / 64 + wave] = any ? tid + 63 - __builtin_clzll(any) : -1;
    }
    __syncthreads();
    // (where rounding leaves no thread past the target: the part's last weight)
    int owner = -1, latest = -1;
    for (int v = kDT / 64 - 1; v >= 0; --v) {
      owner = lds.flags[v] >= 0 ? lds.flags[v] : owner;
      latest = max(latest, lds.flags[kDT / 64 + v]);
    }
    const bool exact = owner >= 0;
    owner = exact ? owner : latest;
    if (per == 1) {                  // the thread's one cell is at hand
      if (tid == owner) {
        int got = -1;
        bool done = false;
#pragma unroll
        for (int e = 0; e < kCell; ++e) {
          run += done ? 0.0 : w[e];
          if (!done && w[e] > 0.0) {
            got = first + e;
            done = exact && run > target;
          }
        }
        lds.found = got;
      }
      __syncthreads();
      return lds.found;
    }
    if (tid == owner) {
      lds.waves[0] = run;
      lds.last = count;
    }
    __syncthreads();
    // the thread's cells, now a lane each (a run of them where they are more)
    const double from = lds.waves[0];
    const int cells = lds.last, each = (cells + 63) / 64;
    const int at = (unit * kDT + owner) * per * kCell + lane * each * kCell;
    const int here = max(0, min(each, cells - lane * each));
    const double sum = weigh_run(row, q, at, kCell, here, weigh, w);
    const double up = wave_scan64(sum);
    const uint64_t in = __builtin_amdgcn_ballot_w64(sum > 0.0 && exact && from + up > target);
    const uint64_t weighty = __builtin_amdgcn_ballot_w64(sum > 0.0);
    const int of = in ? __builtin_ctzll(in) : 63 - __builtin_clzll(weighty);
    int got = -1;
    if (lane == of) {
      double r0 = from + (up - sum);
      bool done = false;
      for (int r = 0; r < here && !done; ++r) {
        if (here > 1) weigh_run(row, q, at + r * kCell, kCell, 1, weigh, w);
#pragma unroll
        for (int e = 0; e < kCell; ++e) {
          r0 += done ? 0.0 : w[e];
          if (!done && w[e] > 0.0) {
            got = at + r * kCell + e;
            done = in && r0 > target;
          }
        }
      }
    }
    return __shfl(got, of, 64);
  }
}

template <typename T, typename Q>
__global__ __launch_bounds__(kDT) void verify_draw_kernel(Verify a) {
  __shared__ DrawLds lds;
  const int seq = blockIdx.x / a.parts, s = blockIdx.x - seq * a.parts, tid = threadIdx.x;
  fill_table(lds.table);
  const Decision d = decide<T, Q>(a, seq, lds);
  int64_t* ids = a.ids + seq * a.width;
  if (s == 0) {
    const int r0 = a.cu[seq];
    for (int j = tid; j < a.width; j += kDT)
      if (j != d.run || d.token >= 0)
        ids[j] = j < d.run ? a.tokens[r0 + 1 + j] : j == d.run ? d.token : -1;
    if (tid == 0) {
      a.accepted[seq] = d.run;
      a.decisions[seq] = d;
    }
  }
  if (d.token >= 0) return;
  // (d.rest: the row's whole sum alone, for the next kernel)
  const int got = draw(a, seq, s, d, reinterpret_cast<const T*>(a.logits) + d.row * a.row_stride,
                       (const Q*)nullptr, 1.0, 0, a.sums + (int64_t)seq * a.units, d.rest ? kSumOnly : kCounted,
                       lds);
  if (got > -2 && tid == 0) ids[d.run] = got < 0 ? d.banned : got;   // (the draft is all there is)
}

template <typename T, typename Q>
__global__ __launch_bounds__(kDT) void verify_rest_kernel(Verify a) {
  __shared__ DrawLds lds;
  const int seq = blockIdx.x / a.parts, s = blockIdx.x - seq * a.parts, tid = threadIdx.x;
  const Decision d = a.decisions[seq];
  if (d.token >= 0 || !d.rest) return;
  fill_table(lds.table);
  const T* row = reinterpret_cast<const T*>(a.logits) + d.row * a.row_stride;
  const Q* q = reinterpret_cast<const Q*>(a.probs) + (int64_t)(d.row - seq) * a.probs_stride;
  const double* const all = a.sums + (int64_t)seq * a.units;
  const double own = (tid & 63) < a.units ? all[tid & 63] : 0.0;   // (every wave the same)
  int got = draw(a, seq, s, d, row, q, 1.0 / wave_sum64(own), 1, a.rest + (int64_t)seq * a.units,
                 kCounted, lds);
  if (got == -2) return;
  if (got == -1)                     // q covers p: from p, by the sums of before
    got = draw(a, seq, s, d, row, (const Q*)nullptr, 1.0, 0, const_cast<double*>(all), kKnown, lds);
  if (tid == 0) a.ids[seq * a.width + d.run] = got;
}

// Workgroups a row of the first kernel: one round of loads where that makes a thousand workgroups, fewer otherwise, at least one.
static int32_t row_splits(int64_t n_rows, int64_t vocab, int eb) {
  const int64_t chunks = vocab * eb / 16;
  const int64_t round = (chunks + kChunks * kVT - 1) / (kChunks * kVT);
  const int64_t want = std::max<int64_t>((1024 + n_rows - 1) / n_rows, round);
  const int64_t most = std::max<int64_t>(chunks / kVT, 1);
  return (int32_t)std::max<int64_t>(std::min<int64_t>({want, most, kMaxSplits}), 1);
}
// A drawn row's units, at most a lane each: a cell a thread of a workgroup, or as many
// as that takes.
static int32_t unit_cells(int64_t vocab) {
  return (int32_t)((vocab + (int64_t)kMaxSplits * kPart - 1) / ((int64_t)kMaxSplits * kPart));
}
static int32_t row_units(int64_t vocab) {
  const int64_t unit = (int64_t)unit_cells(vocab) * kPart;
  return (int32_t)((vocab + unit - 1) / unit);
}
// Parts of a drawn row: about 512 workgroups (two a compute unit; each repeats the
// decision): 64 sequences take 51.4 us, with 256 53.7, with 1024 54.6; a unit each at
// least.
static int32_t seq_parts(int64_t n_seqs, int64_t vocab) {
  return (int32_t)std::min<int64_t>((512 + n_seqs - 1) / n_seqs, row_units(vocab));
}

struct VerifySpace { int64_t stats, decisions, sums, rest, counters, bytes; };
static VerifySpace verify_space(int64_t rows, int64_t seqs, int64_t vocab, int eb) {
  VerifySpace s;
  const int64_t units = row_units(vocab);
  s.stats = 0;
  s.decisions = rows * row_splits(rows, vocab, eb) * (int64_t)sizeof(RowStats);
  s.sums = s.decisions + seqs * (int64_t)sizeof(Decision);
  s.rest = s.sums + seqs * units * 8;
  s.counters = s.rest + seqs * units * 8;
  s.bytes = s.counters + seqs * 2 * 4;
  return s;
}

}  // namespace pkv

using namespace pkv;

extern "C" {

int64_t pkv_verify_workspace_bytes(int64_t n_rows, int64_t n_seqs, int64_t vocab, int32_t dtype) {
  const int eb = elem_bytes(dtype);
  if (!eb || n_rows <= 0 || n_seqs <= 0 || vocab <= 0) return 0;
  return verify_space(n_rows, n_seqs, vocab, eb).bytes;
}

int pkv_verify_drafts(const void* logits, int64_t n_rows, int64_t vocab, int64_t row_stride,
                      int32_t dtype, const int64_t* tokens, const int32_t* cu_query_lens,
                      const int32_t* batch_indices, int64_t n_seqs, const float* numbers,
                      const void* draft_probs, int64_t probs_stride, int32_t probs_dtype,
                      const float* temperatures, float temperature, int64_t* ids, int64_t width,
                      int64_t* accepted, void* workspace, int64_t workspace_bytes, void* stream) {
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(PKV_ERR_INVALID, "dtype=%d is not f16, bf16 or f32", dtype);
  if (vocab <= 0 || vocab > (1 << 30))
    return fail(PKV_ERR_INVALID, "vocab=%lld outside [1, 2^30]", (long long)vocab);
  if (n_seqs <= 0 || n_rows < n_seqs || n_rows > (1 << 24))
    return fail(PKV_ERR_INVALID, "%lld rows of %lld sequences", (long long)n_rows, (long long)n_seqs);
  if (n_rows > 1 && row_stride < vocab)
    return fail(PKV_ERR_INVALID, "row_stride=%lld is shorter than a row of %lld logits",
                (long long)row_stride, (long long)vocab);
  if (draft_probs && !elem_bytes(probs_dtype))
    return fail(PKV_ERR_INVALID, "probs_dtype=%d is not f16, bf16 or f32", probs_dtype);
  if (draft_probs && n_rows - n_seqs > 1 && probs_stride < vocab)
    return fail(PKV_ERR_INVALID, "probs_stride=%lld is shorter than a row of %lld probabilities",
                (long long)probs_stride, (long long)vocab);
  if (width < 1 || width > n_rows)
    return fail(PKV_ERR_INVALID, "width=%lld outside [1, %lld]", (long long)width, (long long)n_rows);
  if (!logits || !tokens || !cu_query_lens || !batch_indices || !numbers || !ids || !accepted ||
      !workspace)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const VerifySpace sp = verify_space(n_rows, n_seqs, vocab, eb);
  if (workspace_bytes < sp.bytes || (uintptr_t)workspace % 16)
    return fail(PKV_ERR_INVALID, "workspace of %lld bytes at %p; %lld, aligned to 16, are needed",
                (long long)workspace_bytes, workspace, (long long)sp.bytes);
  Verify a;
  a.logits = logits;
  a.probs = n_rows > n_seqs ? draft_probs : nullptr;
  a.tokens = tokens;
  a.cu = cu_query_lens;
  a.owner = batch_indices;
  a.numbers = numbers;
  a.temps = temperatures;
  a.stats = (RowStats*)workspace;
  a.decisions = (Decision*)((char*)workspace + sp.decisions);
  a.sums = (double*)((char*)workspace + sp.sums);
  a.rest = (double*)((char*)workspace + sp.rest);
  a.counters = (int32_t*)((char*)workspace + sp.counters);
  a.ids = ids;
  a.accepted = accepted;
  a.row_stride = row_stride;
  a.probs_stride = probs_stride;
  a.width = width;
  a.n_rows = (int32_t)n_rows;
  a.n_seqs = (int32_t)n_seqs;
  a.vocab = (int32_t)vocab;
  a.splits = row_splits(n_rows, vocab, eb);
  a.parts = seq_parts(n_seqs, vocab);
  a.units = row_units(vocab);
  a.cells = unit_cells(vocab);
  a.temp = temperature;
  // terms: an exponent down to -60 (smaller ones add nothing) rounds three times by
  // 2^-24 of itself, the exponential by 2^-22; sums: one rounding a term
  a.error = 0x1p-16f + (float)(vocab / ((int64_t)a.splits * kVT) + 64) * 0x1p-24f;
  hipStream_t s = (hipStream_t)stream;
  const int64_t row_groups = n_rows * a.splits, seq_groups = n_seqs * a.parts;
  if (!launchable(row_groups, kVT) || !launchable(seq_groups, kDT))
    return fail(PKV_ERR_INVALID, "%lld rows of %lld sequences are too many for one call",
                (long long)n_rows, (long long)n_seqs);
  const unsigned rows = (unsigned)row_groups, seqs = (unsigned)seq_groups;
  auto run = [&](auto type, auto probs) -> int {
    typedef decltype(type) T;
    typedef decltype(probs) Q;
    hipLaunchKernelGGL(verify_stats_kernel<T>, dim3(rows), dim3(kVT), 0, s, a);
    PKV_LAUNCH_CHECK();
    hipLaunchKernelGGL((verify_draw_kernel<T, Q>), dim3(seqs), dim3(kDT), 0, s, a);
    PKV_LAUNCH_CHECK();
    if (a.probs) {
      hipLaunchKernelGGL((verify_rest_kernel<T, Q>), dim3(seqs), dim3(kDT), 0, s, a);
      PKV_LAUNCH_CHECK();
    }
    return PKV_OK;
  };
  auto by_probs = [&](auto type) -> int {
    if (!a.probs || probs_dtype == PKV_DTYPE_F32) return run(type, float{});
    return probs_dtype == PKV_DTYPE_F16 ? run(type, _Float16{}) : run(type, __bf16{});
  };
  if (dtype == PKV_DTYPE_F16) return by_probs(_Float16{});
  if (dtype == PKV_DTYPE_BF16) return by_probs(__bf16{});
  return by_probs(float{});
}

}  // extern "C"
