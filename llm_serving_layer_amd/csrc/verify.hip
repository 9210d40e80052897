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
//    error takes the row's sum in 64 bits. The workgroups then sum their part of
//    the one row that a token is drawn from in 64 bits: an exponential is a table
//    of 256 entries in LDS and a polynomial of degree 4, some 20 instructions, on
//    n rows instead of all. The last one to arrive finds the token, except where
//    the row's whole sum is needed first:
//  * verify_rest_kernel, with draft probabilities: the same over max(p - q, 0).
//    In 32 bits the sum's error would move the border of every token behind it.
#include <algorithm>

#include "mfma.h"

namespace pkv {

constexpr int kVT = 256;            // threads of a workgroup
constexpr int kMaxSplits = 64;

struct RowStats { float m, z; int32_t arg, pad; };

struct Verify {
  const void* logits;
  const void* probs;
  const int64_t* tokens;
  const int32_t *cu, *owner;
  const float *numbers, *temps;
  RowStats* stats;
  double *sums, *rest;              // of a sequence's parts: 2^x, max(2^x - q z, 0)
  int32_t* counters;                // two a sequence; cleared by the first kernel
  int64_t *ids, *accepted;
  int64_t row_stride, probs_stride, width;
  int32_t n_rows, n_seqs, vocab, splits, parts;
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

template <typename T>
__global__ __launch_bounds__(kVT) void verify_stats_kernel(Verify a) {
  constexpr int E = 16 / (int)sizeof(T), U = 8;
  typedef T TV __attribute__((ext_vector_type(E)));
  const int r = blockIdx.x / a.splits, s = blockIdx.x - r * a.splits;
  const int tid = threadIdx.x;
  if (s == 0 && r < a.n_seqs && tid < 2) a.counters[2 * r + tid] = 0;
  const T* row = reinterpret_cast<const T*>(a.logits) + r * a.row_stride;
  int begin, end;
  part_of(row, a.vocab, s, a.splits, begin, end);
  const int seq = a.owner[r];
  const float t = a.temps ? (seq >= 0 && seq < a.n_seqs ? a.temps[seq] : 1.f) : a.temp;
  const float c = fminf(kLog2e / (t > 0.f ? t : 1.f), 0x1p100f);
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
#pragma unroll
    for (int u = 0; u < U; ++u) {
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
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e)
          z += __builtin_amdgcn_exp2f(__builtin_fmaf(Elem<T>::to_f(w[u][e]), c, rc));
    } else {                         // (far from 1: the products may overflow)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e)
          z += __builtin_amdgcn_exp2f((Elem<T>::to_f(w[u][e]) - ref) * c);
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
    const int stop = min(ba + E, end);
    for (int i = ba; i < stop; ++i)
      if (Elem<T>::to_f(row[i]) == bm) { ba = i; break; }
  } else {
    ba = begin;                      // (nothing but NaN, or an empty part)
  }
  a.stats[(int64_t)r * a.splits + s] = RowStats{bm, bz, ba, 0};
}

// ------------------------------------------------------------ 64-bit sums ---

// 2^(j / 256)
__device__ __forceinline__ void fill_table(double* table) {
  for (int j = threadIdx.x; j < 256; j += kVT) table[j] = exp2((double)j / 256.0);
  __syncthreads();
}
// 2^x for x <= 0, 0 below -1000 (and for NaN): x = n / 256 + f, |f| <= 2^-9, the
// polynomial's rest below 2^-55.
__device__ __forceinline__ double exp2_64(double x, const double* table) {
  constexpr double kMagic = 6755399441055744.0 / 256.0;   // 1.5 2^52 / 256: adds round to n / 256
  const double at = x + kMagic;
  const double f = (x - (at - kMagic)) * 0.693147180559945309417;
  const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, at);
  double p = __builtin_fma(f, 1.0 / 24.0, 1.0 / 6.0);
  p = __builtin_fma(f, p, 0.5);
  p = __builtin_fma(f, p, 1.0);
  const double base = table[n & 255];
  const double y = __builtin_fma(base * f, p, base);
  const uint64_t bits = __builtin_bit_cast(uint64_t, y) + ((uint64_t)(uint32_t)(n >> 8) << 52);
  return x >= -1000.0 ? __builtin_bit_cast(double, bits) : 0.0;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// the sum over the workgroup, in every thread (4 doubles of LDS)
__device__ __forceinline__ double block_sum64(double v, double* lds) {
  v = wave_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kVT / 64; ++w) s += lds[w];
  return s;
}

// f(index, logit) over elements [begin, end) of a row, 16 bytes at a time; the
// inner borders lie on 16-byte boundaries.
template <typename T, typename F>
__device__ __forceinline__ void each(const T* row, int begin, int end, F&& f) {
  constexpr int E = 16 / (int)sizeof(T);
  typedef T TV __attribute__((ext_vector_type(E)));
  const int head = min((int)((-(uintptr_t)(row + begin) & 15) / sizeof(T)), end - begin);
  const int body = begin + head, chunks = (end - body) / E, tail = body + chunks * E;
  if ((int)threadIdx.x < head) f(begin + threadIdx.x, Elem<T>::to_f(row[begin + threadIdx.x]));
  for (int k = threadIdx.x; k < chunks; k += kVT) {
    const TV w = *reinterpret_cast<const TV*>(row + body + (int64_t)k * E);
#pragma unroll
    for (int e = 0; e < E; ++e) f(body + k * E + e, Elem<T>::to_f(w[e]));
  }
  if (tail + (int)threadIdx.x < end)
    f(tail + threadIdx.x, Elem<T>::to_f(row[tail + threadIdx.x]));
}

// A sequence's decision: how many drafts stand, and the row that follows.
struct Decision {
  int run, row, token;     // token: taken as it is, or -1: drawn from the row
  int banned;              // the draft that fell, without draft probabilities; -1
  bool rest;               // drawn from max(p - q, 0)
  double m, c;             // the row's largest logit, log2 e / temperature
};

// (uniform over the workgroup; lds: 4 doubles, flags: kVT ints)
template <typename T, typename Q>
__device__ Decision decide(const Verify& a, int seq, const double* table, double* lds, int* flags) {
  const int r0 = a.cu[seq], n = a.cu[seq + 1] - r0;
  const float t = a.temps ? a.temps[seq] : a.temp;
  const bool greedy = !(t > 0.f);
  const double c = 1.44269504088896340736 / (greedy ? 1.0 : (double)t);
  const T* logits = reinterpret_cast<const T*>(a.logits);
  const int tid = threadIdx.x;
  auto whole = [&](int r) {          // a row's statistics
    const RowStats* st = a.stats + (int64_t)r * a.splits;
    RowStats b = st[0];
    for (int s = 1; s < a.splits; ++s) b.m = fmaxf(b.m, st[s].m);
    b.z = 0.f;
    b.arg = 0x7fffffff;
    const float ref = b.m == -INFINITY ? 0.f : b.m;
    for (int s = 0; s < a.splits; ++s) {
      b.z += st[s].z * __builtin_amdgcn_exp2f((st[s].m - ref) * fminf((float)c, 0x1p100f));
      if (st[s].m == b.m) b.arg = min(b.arg, st[s].arg);
    }
    return b;
  };
  Decision d;
  d.c = c;
  d.run = n - 1;
  for (int j0 = 0; j0 < n - 1; j0 += kVT) {
    const int j = j0 + tid;
    int state = 1;                   // 0: falls, 1: stands, 2: too close to tell
    if (j < n - 1) {
      const int r = r0 + j;
      const int64_t x = a.tokens[r + 1];
      const RowStats b = whole(r);
      if (x < 0 || x >= a.vocab) {
        state = 0;
      } else if (greedy) {
        state = b.z == b.z && b.arg == x;
      } else {
        const double qx =
            a.probs ? (double)Elem<Q>::to_f(
                          reinterpret_cast<const Q*>(a.probs)[(int64_t)(r - seq) * a.probs_stride + x])
                    : 1.0;
        const double ex = exp2_64(
            ((double)Elem<T>::to_f(logits[r * a.row_stride + x]) - (double)b.m) * c, table);
        const double need = (double)a.numbers[r] * qx * (double)b.z;
        // the sum's error, relative: its terms' and their sums' (a.error), and what
        // the rounding of m c does to every exponent
        const double error = (double)a.error + fmin(fabs((double)b.m * c), 0x1p80) * 0x1p-23;
        state = need < ex;
        if (fabs(need - ex) <= error * fabs(need)) state = 2;
        if (!(b.z == b.z)) state = 0;
      }
    }
    flags[tid] = state;
    __syncthreads();
    int stop = min(kVT, n - 1 - j0);
    for (int i = 0; i < stop; ++i) {
      int s = flags[i];
      if (s == 1) continue;
      if (s == 2) {                  // the row's sum in 64 bits
        const int r = r0 + j0 + i;
        const T* row = logits + r * a.row_stride;
        const RowStats b = whole(r);
        double z = 0.0;
        each(row, 0, a.vocab, [&](int, float l) { z += exp2_64(((double)l - (double)b.m) * c, table); });
        z = block_sum64(z, lds);
        const int64_t x = a.tokens[r + 1];
        const double qx =
            a.probs ? (double)Elem<Q>::to_f(
                          reinterpret_cast<const Q*>(a.probs)[(int64_t)(r - seq) * a.probs_stride + x])
                    : 1.0;
        const double ex = exp2_64(((double)Elem<T>::to_f(row[x]) - (double)b.m) * c, table);
        if ((double)a.numbers[r] * qx < ex / z) continue;
      }
      d.run = j0 + i;
      break;
    }
    __syncthreads();                 // flags are free again
    if (d.run < n - 1) break;
  }
  d.row = r0 + d.run;
  const RowStats b = whole(d.row);
  d.m = b.m;
  d.token = -1;
  const bool none = !(b.z == b.z) || b.m == -INFINITY;   // no distribution
  if (greedy || none) d.token = b.arg;
  if (!(b.z == b.z)) {               // a NaN, or +inf: torch's order, the first NaN first
    if (tid == 0) flags[0] = 0x7fffffff;
    __syncthreads();
    each(logits + d.row * a.row_stride, 0, a.vocab, [&](int i, float l) {
      if (l != l) atomicMin(&flags[0], i);
    });
    __syncthreads();
    if (flags[0] != 0x7fffffff) d.token = flags[0];
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

struct DrawLds {
  double table[256];
  double sums[kVT];
  double four[kVT / 64];
  int flags[kVT];
  int last, found, any;
};

// The token of a sequence from its parts' sums (sums[0 .. parts)), in the
// workgroup that arrived last: the part, then the thread, then the element whose
// running sum passes the target. weight(index): an element's weight.
template <typename T, typename F>
__device__ int pick(const Verify& a, int seq, const T* row, const double* sums, DrawLds& lds,
                    F&& weight) {
  const int tid = threadIdx.x;
  const float u = a.numbers[a.cu[seq + 1] - 1];
  double total = 0.0;
  for (int s = 0; s < a.parts; ++s) total += sums[s];
  const double target = (double)u * total;
  double base = 0.0;
  int part = -1, lastp = 0;
  for (int s = 0; s < a.parts; ++s) {
    if (sums[s] > 0.0) lastp = s;
    if (base + sums[s] > target) { part = s; break; }
    base += sums[s];
  }
  if (part < 0) {                    // (a number of 1, or the last sum's rounding)
    part = lastp;
    base = INFINITY;
  }
  int begin, end;
  part_of(row, a.vocab, part, a.parts, begin, end);
  const int per = (end - begin + kVT - 1) / kVT;
  const int b = min(begin + tid * per, end), e = min(b + per, end);
  double mine = 0.0;
  for (int i = b; i < e; ++i) mine += weight(i);
  __syncthreads();
  lds.sums[tid] = mine;
  if (tid == 0) {
    lds.found = 0x7fffffff;
    lds.any = -1;
  }
  __syncthreads();
  double before = base;
  for (int i = 0; i < tid; ++i) before += lds.sums[i];
  if (before + mine > target && base < INFINITY) atomicMin(&lds.found, tid);
  if (mine > 0.0) atomicMax(&lds.any, tid);
  __syncthreads();
  // (where rounding leaves no thread past the target: the part's last weight)
  const bool exact = lds.found != 0x7fffffff;
  const int owner = exact ? lds.found : lds.any;
  __syncthreads();
  if (tid == owner) {
    int got = -1;
    double run = before;
    for (int i = b; i < e; ++i) {
      const double w = weight(i);
      run += w;
      if (w > 0.0) got = i;
      if (exact && run > target && w > 0.0) break;
    }
    lds.found = got;
  }
  __syncthreads();
  const int out = owner < 0 ? -1 : lds.found;
  __syncthreads();
  return out;
}

// Whether this workgroup is the last of its sequence to arrive at counter k; its
// part's sum is stored where the last one reads all of them. (Stores and loads
// beyond the XCDs' caches; the wait before the count.)
__device__ __forceinline__ bool arrive(const Verify& a, int seq, int k, double* at, double sum,
                                       DrawLds& lds) {
  if (threadIdx.x == 0) {
    __hip_atomic_store(at, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds.last = __hip_atomic_fetch_add(a.counters + 2 * seq + k, 1, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) == a.parts - 1;
  }
  __syncthreads();
  return lds.last;
}
// a sequence's sums into lds.sums, by the last one to arrive
__device__ __forceinline__ void read_sums(const Verify& a, const double* sums, DrawLds& lds) {
  __syncthreads();
  for (int s = threadIdx.x; s < a.parts; s += kVT)
    lds.sums[s] = __hip_atomic_load(sums + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
}

template <typename T, typename Q>
__global__ __launch_bounds__(kVT) void verify_draw_kernel(Verify a) {
  __shared__ DrawLds lds;
  __shared__ double parts[kMaxSplits];
  const int seq = blockIdx.x / a.parts, s = blockIdx.x - seq * a.parts, tid = threadIdx.x;
  fill_table(lds.table);
  const Decision d = decide<T, Q>(a, seq, lds.table, lds.four, lds.flags);
  int64_t* ids = a.ids + seq * a.width;
  if (s == 0) {
    const int r0 = a.cu[seq];
    for (int j = tid; j < a.width; j += kVT)
      if (j != d.run || d.token >= 0) ids[j] = j < d.run ? a.tokens[r0 + 1 + j] : j == d.run ? d.token : -1;
    if (tid == 0) a.accepted[seq] = d.run;
  }
  if (d.token >= 0) return;
  const T* row = reinterpret_cast<const T*>(a.logits) + d.row * a.row_stride;
  int begin, end;
  part_of(row, a.vocab, s, a.parts, begin, end);
  double sum = 0.0;
  each(row, begin, end, [&](int i, float l) {
    const double w = exp2_64(((double)l - d.m) * d.c, lds.table);
    sum += i == d.banned ? 0.0 : w;
  });
  sum = block_sum64(sum, lds.four);
  double* const sums = a.sums + (int64_t)seq * a.parts;
  if (d.rest) {                      // the row's whole sum, for the next kernel
    if (tid == 0) sums[s] = sum;
    return;
  }
  if (!arrive(a, seq, 0, sums + s, sum, lds)) return;
  read_sums(a, sums, lds);
  for (int i = tid; i < a.parts; i += kVT) parts[i] = lds.sums[i];
  __syncthreads();
  const int got = pick(a, seq, row, parts, lds, [&](int i) {
    return i == d.banned ? 0.0
                         : exp2_64(((double)Elem<T>::to_f(row[i]) - d.m) * d.c, lds.table);
  });
  if (tid == 0) ids[d.run] = got < 0 ? d.banned : got;   // (the draft is all there is)
}

template <typename T, typename Q>
__global__ __launch_bounds__(kVT) void verify_rest_kernel(Verify a) {
  __shared__ DrawLds lds;
  __shared__ double parts[kMaxSplits];
  const int seq = blockIdx.x / a.parts, s = blockIdx.x - seq * a.parts, tid = threadIdx.x;
  fill_table(lds.table);
  const Decision d = decide<T, Q>(a, seq, lds.table, lds.four, lds.flags);
  if (d.token >= 0 || !d.rest) return;
  const T* row = reinterpret_cast<const T*>(a.logits) + d.row * a.row_stride;
  const Q* qrow = reinterpret_cast<const Q*>(a.probs) + (int64_t)(d.row - seq) * a.probs_stride;
  const double* const all = a.sums + (int64_t)seq * a.parts;
  double z = 0.0;
  for (int i = 0; i < a.parts; ++i) z += all[i];
  const double iz = 1.0 / z;
  auto weight = [&](int i, float l) {
    const double w = exp2_64(((double)l - d.m) * d.c, lds.table) * iz - (double)Elem<Q>::to_f(qrow[i]);
    return w > 0.0 ? w : 0.0;
  };
  int begin, end;
  part_of(row, a.vocab, s, a.parts, begin, end);
  double sum = 0.0;
  each(row, begin, end, [&](int i, float l) { sum += weight(i, l); });
  sum = block_sum64(sum, lds.four);
  double* const rest = a.rest + (int64_t)seq * a.parts;
  if (!arrive(a, seq, 1, rest + s, sum, lds)) return;
  read_sums(a, rest, lds);
  for (int i = tid; i < a.parts; i += kVT) parts[i] = lds.sums[i];
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < a.parts; ++i) total += parts[i];
  int got;
  if (total > 0.0) {
    got = pick(a, seq, row, parts, lds,
               [&](int i) { return weight(i, Elem<T>::to_f(row[i])); });
  } else {                           // q covers p: from p
    __syncthreads();
    for (int i = tid; i < a.parts; i += kVT) parts[i] = all[i];
    __syncthreads();
    got = pick(a, seq, row, parts, lds, [&](int i) {
      return exp2_64(((double)Elem<T>::to_f(row[i]) - d.m) * d.c, lds.table);
    });
  }
  if (tid == 0) a.ids[seq * a.width + d.run] = got;
}

// Workgroups a row of the first kernel: about 2048 of them, at most 8 chunks of 16
// bytes a thread (one round of loads) where there are enough rows, at least one.
static int32_t row_splits(int64_t n_rows, int64_t vocab, int eb) {
  const int64_t chunks = vocab * eb / 16;
  const int64_t want = std::max<int64_t>((2048 + n_rows - 1) / n_rows, 1);
  const int64_t most = std::max<int64_t>(chunks / kVT, 1);
  return (int32_t)std::min<int64_t>({want, most, kMaxSplits});
}
// Parts of a drawn row: about 1024 workgroups, at least 8 elements a thread.
static int32_t seq_parts(int64_t n_seqs, int64_t vocab) {
  const int64_t want = std::max<int64_t>((1024 + n_seqs - 1) / n_seqs, 1);
  const int64_t most = std::max<int64_t>(vocab / (8 * kVT), 1);
  return (int32_t)std::min<int64_t>({want, most, kMaxSplits});
}

struct VerifySpace { int64_t stats, sums, rest, counters, bytes; };
static VerifySpace verify_space(int64_t rows, int64_t seqs, int64_t vocab, int eb) {
  VerifySpace s;
  const int64_t parts = seq_parts(seqs, vocab);
  s.stats = 0;
  s.sums = rows * row_splits(rows, vocab, eb) * (int64_t)sizeof(RowStats);
  s.rest = s.sums + seqs * parts * 8;
  s.counters = s.rest + seqs * parts * 8;
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
  a.temp = temperature;
  // terms: an exponent down to -60 (smaller ones add nothing) rounds three times by
  // 2^-24 of itself, the exponential by 2^-22; sums: one rounding a term
  a.error = 0x1p-16f + (float)(vocab / ((int64_t)a.splits * kVT) + 64) * 0x1p-24f;
  hipStream_t s = (hipStream_t)stream;
  const unsigned rows = (unsigned)(n_rows * a.splits), seqs = (unsigned)(n_seqs * a.parts);
  auto run = [&](auto type, auto probs) -> int {
    typedef decltype(type) T;
    typedef decltype(probs) Q;
    hipLaunchKernelGGL(verify_stats_kernel<T>, dim3(rows), dim3(kVT), 0, s, a);
    PKV_LAUNCH_CHECK();
    hipLaunchKernelGGL((verify_draw_kernel<T, Q>), dim3(seqs), dim3(kVT), 0, s, a);
    PKV_LAUNCH_CHECK();
    if (a.probs) {
      hipLaunchKernelGGL((verify_rest_kernel<T, Q>), dim3(seqs), dim3(kVT), 0, s, a);
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
