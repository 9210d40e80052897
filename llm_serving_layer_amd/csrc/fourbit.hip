// The 4-bit cache's rows: append (quantise), read (the values held), and
// attention over it for any geometry. The format is fourbit.h's.
#include <algorithm>
#include <type_traits>

#include "fourbit.h"

namespace pkv {

// ----------------------------------------------------------------- append ---

// A tiled row group (64 elements) by 8 lanes of 8 elements: 16-byte loads, a minimum
// and maximum over the 8 lanes, then each lane's codes: K one word, V four bytes.
// Its inputs are 4 of 5 bytes that it moves; what bounds it is the vector work: a group's
// elements next to a border between codes are looked for together and all decided in
// 64 bits where there is one (a wave in 16), codes are packed as sums in float.
// 5 to 6 thousand tokens of 8 heads of 128 (32 MB) take 14.4 us, 2.2 TB/s: 284 vector
// instructions a wave are 11 of them, the ramps of a short launch (one token: 2.3) the rest.
template <typename T>
__global__ __launch_bounds__(256) void append_4bit_kernel(
    unsigned char* __restrict__ kpool, unsigned char* __restrict__ vpool, int64_t num_slots,
    FourBit f, Div by_row, Div by_group, Div by_page, const T* __restrict__ k, int64_t k_stride,
    const T* __restrict__ v, int64_t v_stride, const int32_t* __restrict__ slots, uint32_t total,
    int32_t* status) {
  const uint32_t unit = blockIdx.x * 32 + (threadIdx.x >> 3);
  const bool live = unit < total;
  uint32_t hq, r;
  const uint32_t row = divide(live ? unit : total - 1, by_row, hq);   // (token, K or V)
  const uint32_t t = row >> 1;
  const bool is_v = row & 1;
  const int l = threadIdx.x & 7;
  const int32_t slot = slots[t];
  typedef T TV __attribute__((ext_vector_type(8)));
  // (heads lie one after another, so group hq of the row starts at 64 hq)
  const TV in = *reinterpret_cast<const TV*>((is_v ? v + t * v_stride : k + t * k_stride) +
                                             hq * 64 + l * 8);
  float x[8], lo = INFINITY, hi = -INFINITY, finite = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = Elem<T>::to_f(in[i]);
    finite = __builtin_fmaf(x[i], 0.f, finite);           // (NaN of an infinity or NaN)
    if constexpr (!std::is_same<T, _Float16>::value)
      x[i] = __builtin_amdgcn_fmed3f(x[i], -kF16Max, kF16Max);
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
  lo = fminf(lo, dpp<0xB1>(lo));     // quad_perm [1,0,3,2]
  hi = fmaxf(hi, dpp<0xB1>(hi));
  lo = fminf(lo, dpp<0x4E>(lo));     // quad_perm [2,3,0,1]
  hi = fmaxf(hi, dpp<0x4E>(hi));
  lo = fminf(lo, dpp<0x141>(lo));    // row_half_mirror: the 8 lanes
  hi = fmaxf(hi, dpp<0x141>(hi));
  const uint64_t odds = __builtin_amdgcn_ballot_w64(finite != 0.f);
  const bool none = (odds >> (threadIdx.x & 56)) & 0xffu;
  const uint32_t pair = none ? kNanPair : group_pair(none ? 0.f : lo, none ? 0.f : hi);
  const float step = none ? 0.f : pair_step(pair), zero = none ? 0.f : pair_zero(pair);
  const float inv = step > 0.f ? 1.f / step : 0.f;
  // Codes: off by less than 2^-17 of a step, so wrong only next to a border; 15 steps
  // reach the largest element, so none passes 15.
  float c[8], far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w = (x[i] - zero) * inv;
    c[i] = __builtin_rintf(w);
    far = fmaxf(far, __builtin_fabsf(w - c[i]));
  }
  if (__builtin_amdgcn_ballot_w64(far > 0.5f - 0x1p-14f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = (float)code_of(x[i], step, inv, zero);
  }
  if (none) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 0.f;
  }
  const uint32_t block = divide((uint32_t)slot, by_page, r);
  const bool write = live && slot >= 0 && slot < num_slots;
  if (live && !write && hq == 0 && l == 0) flag(status, PKV_STATUS_BAD_SLOT);
  unsigned char* const base = (is_v ? vpool : kpool) + (int64_t)block * f.block;
  uint32_t q;
  const uint32_t h = divide(hq, by_group, q);
  unsigned char* const codes = base + h * f.head_bytes;
  if (write && l == 0) reinterpret_cast<uint32_t*>(base + f.pairs)[hq * f.ps + r] = pair;
  if (!is_v) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float four = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(c[i + 3], 16.f, c[i + 2]),
                                                       16.f, c[i + 1]), 16.f, c[i]);
      w |= (uint32_t)four << (4 * i);
    }
    if (write) *reinterpret_cast<uint32_t*>(codes + k_byte(f, r, q * 64 + l * 8)) = w;
  }
  if (__builtin_amdgcn_ballot_w64(is_v)) {
    // Dims 32 b + n and 32 b + 16 + n share a byte: lanes two apart. Lanes (l & 2) == 0
    // hold dims n, the others n + 16; each writes four of the pair's eight bytes.
    const bool upper = l & 2;
    uint32_t bytes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float own = upper ? c[4 + i] : c[i], sent = dpp<0x4E>(upper ? c[i] : c[4 + i]);
      const float byte = upper ? __builtin_fmaf(own, 16.f, sent) : __builtin_fmaf(sent, 16.f, own);
      bytes = __builtin_amdgcn_cvt_pk_u8_f32(byte, i, bytes);
    }
    if (!write || !is_v) return;
    unsigned char* const to =
        codes + v_byte(f, r, q * 64 + (l >> 2) * 32 + (l & 1) * 8 + (upper ? 4 : 0));
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i * (f.d / 8)] = (unsigned char)(bytes >> (8 * i));
  }
}

// Any geometry: a wave per (token, K or V, head), one group.
template <typename T>
__global__ __launch_bounds__(64) void append_4bit_any_kernel(
    unsigned char* __restrict__ kpool, unsigned char* __restrict__ vpool, int64_t num_slots,
    FourBit f, const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
    int64_t v_stride, const int32_t* __restrict__ slots, int32_t* status) {
  const int64_t row = blockIdx.x / f.n_kv;
  const int h = (int)(blockIdx.x - row * f.n_kv);
  const int64_t t = row >> 1;
  const bool is_v = row & 1;
  const int lane = threadIdx.x;
  const int64_t slot = slots[t];
  if (slot < 0 || slot >= num_slots) {
    if (h == 0 && lane == 0) flag(status, PKV_STATUS_BAD_SLOT);
    return;
  }
  const T* src = (is_v ? v + t * v_stride : k + t * k_stride) + (int64_t)h * f.d;
  const int64_t block = slot / f.ps;
  const int r = (int)(slot - block * f.ps);
  unsigned char* base = (is_v ? vpool : kpool) + block * f.block;
  const int size = f.d / f.groups;
  for (int q = 0; q < f.groups; ++q) {
    float lo = INFINITY, hi = -INFINITY;
    bool odd = false;
    for (int i = lane; i < size; i += 64) {
      float x = Elem<T>::to_f(src[q * size + i]);
      odd |= !(__builtin_fabsf(x) < INFINITY);
      x = fminf(fmaxf(x, -kF16Max), kF16Max);
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
    }
    const bool none = __builtin_amdgcn_ballot_w64(odd) != 0;
    lo = -wave_max(-lo);
    hi = wave_max(hi);
    const uint32_t pair = none ? kNanPair : group_pair(lo, hi);
    const float step = none ? 0.f : pair_step(pair), zero = pair_zero(pair), inv = 1.f / step;
    if (lane == 0)
      reinterpret_cast<uint32_t*>(base + f.pairs)[(h * f.groups + q) * f.ps + r] = pair;
    for (int i = lane; i < size / 2; i += 64) {   // a byte: elements a and b
      const int a = f.tiled && is_v ? (i / 16) * 32 + i % 16 : 2 * i;
      const int b = f.tiled && is_v ? a + 16 : a + 1;
      uint32_t c[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = Elem<T>::to_f(src[q * size + (j ? b : a)]);
        x = fminf(fmaxf(x, -kF16Max), kF16Max);
        c[j] = code_of(x, step, inv, zero);
      }
      const int e = q * size + a;
      base[h * f.head_bytes + (is_v ? v_byte(f, r, e) : k_byte(f, r, e))] =
          (unsigned char)(c[0] | c[1] << 4);
    }
  }
}

// ------------------------------------------------------------------- read ---

// The values that slots hold, rounded once to the pool's type. Tiled: 16 elements a
// thread, K's as two words, V's as the bytes of dims 32 b + n .. + 7 with those 16
// further. Bound by what it writes where there are many rows: 32 MB in 10.6 us, 3
// TB/s, of which a launch's ramps are 2.
template <typename T>
__global__ __launch_bounds__(256) void read_4bit_kernel(
    const unsigned char* __restrict__ kpool, const unsigned char* __restrict__ vpool,
    int64_t num_slots, FourBit f, Div by_row, Div by_head, Div by_page,
    const int32_t* __restrict__ slots, uint32_t total, T* __restrict__ k, T* __restrict__ v,
    int32_t* status) {
  typedef T TV __attribute__((ext_vector_type(8)));
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  uint32_t at, part, r;                                   // of a row, of a head
  const uint32_t row = divide(i, by_row, at), h = divide(at, by_head, part);
  const uint32_t t = row >> 1;
  const bool is_v = row & 1;
  const int32_t slot = slots[t];
  TV lo{}, hi{};
  if (slot < 0 || slot >= num_slots) {
    if (at == 0) flag(status, PKV_STATUS_BAD_SLOT);
  } else {
    const uint32_t block = divide((uint32_t)slot, by_page, r);
    const unsigned char* base = (is_v ? vpool : kpool) + (int64_t)block * f.block;
    const unsigned char* codes = base + h * f.head_bytes;
    const uint32_t pair =
        reinterpret_cast<const uint32_t*>(base + f.pairs)[(h * f.groups + (part >> 2)) * f.ps + r];
    uint32_t low[2], up[2];       // bytes of the first 8 elements, of the others
    if (is_v) {
      const unsigned char* from = codes + v_byte(f, r, 32 * (part >> 1) + 8 * (part & 1));
      low[0] = low[1] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) low[j >> 2] |= (uint32_t)from[j * (f.d / 8)] << (8 * (j & 3));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        up[j] = low[j] >> 4 & 0x0f0f0f0fu;
        low[j] &= 0x0f0f0f0fu;
      }
    } else {
      const uint32_t* from = reinterpret_cast<const uint32_t*>(codes + k_byte(f, r, 16 * part));
      auto bytes = [](uint32_t w, uint32_t (&of)[2]) {
        const uint32_t even = w & 0x0f0f0f0fu, odd = w >> 4 & 0x0f0f0f0fu;
        of[0] = __builtin_amdgcn_perm(odd, even, 0x05010400u);
        of[1] = __builtin_amdgcn_perm(odd, even, 0x07030602u);
      };
      bytes(from[0], low);
      bytes(from[1], up);
    }
    const float step = pair_step(pair), zero = pair_zero(pair);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = Elem<T>::from_f(
          __builtin_fmaf((float)(low[j >> 2] >> (8 * (j & 3)) & 0xffu), step, zero));
      hi[j] = Elem<T>::from_f(
          __builtin_fmaf((float)(up[j >> 2] >> (8 * (j & 3)) & 0xffu), step, zero));
    }
  }
  // (K: 16 elements in a row; V: 8 and the 8 that lie 16 further)
  T* to = (is_v ? v : k) + (int64_t)t * f.n_kv * f.d + h * f.d +
          (is_v ? 32 * (part >> 1) + 8 * (part & 1) : 16 * part);
  *reinterpret_cast<TV*>(to) = lo;
  *reinterpret_cast<TV*>(to + (is_v ? 16 : 8)) = hi;
}

// Any geometry: two elements a thread.
template <typename T>
__global__ __launch_bounds__(256) void read_4bit_any_kernel(
    const unsigned char* __restrict__ kpool, const unsigned char* __restrict__ vpool,
    int64_t num_slots, FourBit f, Div by_row, Div by_head, Div by_page,
    const int32_t* __restrict__ slots, uint32_t total, T* __restrict__ k, T* __restrict__ v,
    int32_t* status) {
  typedef T TV __attribute__((ext_vector_type(2)));
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  uint32_t at, e, r;
  const uint32_t row = divide(i, by_row, at), h = divide(at, by_head, e);
  const uint32_t t = row >> 1;
  const bool is_v = row & 1;
  e *= 2;
  const int32_t slot = slots[t];
  TV out{};
  if (slot < 0 || slot >= num_slots) {
    if (at == 0) flag(status, PKV_STATUS_BAD_SLOT);
  } else {
    const uint32_t block = divide((uint32_t)slot, by_page, r);
    const unsigned char* base = (is_v ? vpool : kpool) + (int64_t)block * f.block;
    const unsigned char* codes = base + h * f.head_bytes;
    const uint32_t pair =
        reinterpret_cast<const uint32_t*>(base + f.pairs)[(h * f.groups + group_of(f, e)) * f.ps + r];
    const float step = pair_step(pair), zero = pair_zero(pair);
    const int b = codes[is_v ? v_byte(f, r, e) : k_byte(f, r, e)];
    out[0] = Elem<T>::from_f(__builtin_fmaf((float)(b & 15), step, zero));
    out[1] = Elem<T>::from_f(__builtin_fmaf((float)(b >> 4), step, zero));
  }
  *reinterpret_cast<TV*>((is_v ? v : k) + (int64_t)t * f.n_kv * f.d + 2 * at) = out;
}

// ------------------------------------------------ attention, any geometry ---

// One wave per (query token, query head), 64 keys at a time: a lane a key for
// the scores, a lane up to four dims for the values, the running maximum and sum
// between. Everything in 32 bits. Slow by design: for geometries without a
// matrix-core kernel.
template <typename T>
__global__ __launch_bounds__(64) void attend_4bit_any_kernel(
    const T* __restrict__ q, T* __restrict__ out, const unsigned char* __restrict__ kpool,
    const unsigned char* __restrict__ vpool, int64_t num_blocks, FourBit f,
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ indptr,
    const int32_t* __restrict__ indices, const int32_t* __restrict__ kv_lens,
    const int32_t* __restrict__ batch_idx, int32_t n_seqs, int32_t n_heads, float scale_log2,
    int32_t* status) {
  __shared__ float qs[256];
  __shared__ float ps[64];
  __shared__ int32_t page_of[64];
  const int lane = threadIdx.x;
  const int tok = blockIdx.x / n_heads, hq = blockIdx.x - tok * n_heads;
  const int h = hq / (n_heads / f.n_kv);
  const int seq = batch_idx[tok];
  if (seq < 0 || seq >= n_seqs) return;
  const int q0 = cu_q[seq], q_len = cu_q[seq + 1] - q0;
  // keys this token sees (no more than there are, for a token of another sequence)
  const int limit = min(kv_lens[seq] - q_len + (tok - q0) + 1, kv_lens[seq]);
  const int first_page = indptr[seq];
  const T* qr = q + ((int64_t)tok * n_heads + hq) * f.d;
  for (int i = lane; i < f.d; i += 64) qs[i] = Elem<T>::to_f(qr[i]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t0 = 0; t0 < limit; t0 += 64) {
    const int t = t0 + lane;
    const bool in = t < limit;
    float s = -INFINITY;
    int id = -1;
    if (in) {
      id = indices[first_page + t / f.ps];
      s = 0.f;
      if (id < 0 || id >= num_blocks) {
        flag(status, PKV_STATUS_BAD_PAGE);
        id = -1;                                     // read as zeros
      } else {
        const int r = t % f.ps;
        const unsigned char* base = kpool + (int64_t)id * f.block;
        const uint32_t* words =
            reinterpret_cast<const uint32_t*>(base + f.pairs) + h * f.groups * f.ps + r;
        for (int e = 0; e < f.d; e += 2) {           // (a byte of K: two elements)
          const uint32_t w = words[group_of(f, e) * f.ps];
          const int b = base[h * f.head_bytes + k_byte(f, r, e)];
          const float st = pair_step(w), z = pair_zero(w);
          s += qs[e] * __builtin_fmaf((float)(b & 15), st, z);
          s += qs[e + 1] * __builtin_fmaf((float)(b >> 4), st, z);
        }
      }
      s *= scale_log2;
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float p = in ? __builtin_amdgcn_exp2f(s - ref) : 0.f;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);     // (0 at first)
    m = m_new;
    l = l * alpha + wave_sum(p);
    __syncthreads();
    ps[lane] = p;
    page_of[lane] = id;
    __syncthreads();
    const int n = min(64, limit - t0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = lane + 64 * j;
      if (e >= f.d) break;
      float acc = 0.f;
      for (int i = 0; i < n; ++i) {
        if (page_of[i] < 0) continue;
        const int r = (t0 + i) % f.ps;
        const unsigned char* base = vpool + (int64_t)page_of[i] * f.block;
        const uint32_t w = reinterpret_cast<const uint32_t*>(
            base + f.pairs)[(h * f.groups + group_of(f, e)) * f.ps + r];
        const int b = base[h * f.head_bytes + v_byte(f, r, e)];
        acc += ps[i] * __builtin_fmaf((float)(b >> (4 * v_half(f, e)) & 15), pair_step(w),
                                      pair_zero(w));
      }
      o[j] = o[j] * alpha + acc;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = lane + 64 * j;
    if (e < f.d) out[((int64_t)tok * n_heads + hq) * f.d + e] = Elem<T>::from_f(o[j] / l);
  }
}

int check_4bit(int32_t n_kv, int32_t d, int32_t ps) {
  if (n_kv <= 0 || d <= 0 || ps <= 0) return fail(PKV_ERR_INVALID, "non-positive geometry");
  if (d > 256 || d % 2) return fail(PKV_ERR_INVALID, "head_dim=%d is odd or above 256", d);
  if ((int64_t)n_kv * ps * d > (1ll << 30))
    return fail(PKV_ERR_INVALID, "a block of %d x %d x %d elements is too large", ps, n_kv, d);
  return PKV_OK;
}

}  // namespace pkv

using namespace pkv;

extern "C" {

int64_t pkv_block_bytes_4bit(int32_t n_kv_heads, int32_t head_dim, int32_t page_size) {
  if (check_4bit(n_kv_heads, head_dim, page_size)) return 0;
  return four_bit(n_kv_heads, head_dim, page_size).block;
}

int pkv_append_4bit(void* k_pool, void* v_pool, int64_t num_blocks, const void* k,
                    int64_t k_stride, const void* v, int64_t v_stride,
                    const int32_t* slot_mapping, int64_t n_tokens, int32_t n_kv_heads,
                    int32_t head_dim, int32_t page_size, int32_t dtype, int32_t* status_word,
                    void* stream) {
  const int rc = check_4bit(n_kv_heads, head_dim, page_size);
  if (rc) return rc;
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(PKV_ERR_INVALID, "unsupported dtype code %d", dtype);
  if (n_tokens < 0 || num_blocks < 0) return fail(PKV_ERR_INVALID, "negative count");
  if (n_tokens == 0) return PKV_OK;
  if (!k_pool || !v_pool || !k || !v || !slot_mapping)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const FourBit f = four_bit(n_kv_heads, head_dim, page_size);
  hipStream_t s = (hipStream_t)stream;
  const bool wide = f.tiled && ((uintptr_t)k | (uintptr_t)v | (uint64_t)(k_stride * eb) |
                                (uint64_t)(v_stride * eb)) % 16 == 0;
  const int64_t work = n_tokens > 0x7fffffffLL ? n_tokens : n_tokens * 2 * f.n_kv * f.groups;
  if (work > 0x7fffffffLL || !(wide ? launchable((work + 31) / 32, 256)
                                    : launchable(n_tokens * 2 * f.n_kv, 64)))
    return fail(PKV_ERR_INVALID, "too many rows in one append");
  auto go = [&](auto type) {
    typedef decltype(type) T;
    if (wide)
      hipLaunchKernelGGL(append_4bit_kernel<T>, dim3((unsigned)((work + 31) / 32)), dim3(256), 0, s,
                         (unsigned char*)k_pool, (unsigned char*)v_pool, num_blocks * page_size, f,
                         div_by(f.n_kv * f.groups), div_by(f.groups), div_by(page_size),
                         (const T*)k, k_stride,
                         (const T*)v, v_stride, slot_mapping, (uint32_t)work, status_word);
    else
      hipLaunchKernelGGL(append_4bit_any_kernel<T>, dim3((unsigned)(n_tokens * 2 * f.n_kv)), dim3(64), 0, s,
                         (unsigned char*)k_pool, (unsigned char*)v_pool, num_blocks * page_size, f,
                         (const T*)k, k_stride, (const T*)v, v_stride, slot_mapping, status_word);
  };
  if (dtype == PKV_DTYPE_F16) go(_Float16{});
  else if (dtype == PKV_DTYPE_BF16) go(__bf16{});
  else go(float{});
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

int pkv_read_4bit(const void* k_pool, const void* v_pool, int64_t num_blocks,
                  const int32_t* slots, int64_t n_rows, void* k, void* v, int32_t n_kv_heads,
                  int32_t head_dim, int32_t page_size, int32_t dtype, int32_t* status_word,
                  void* stream) {
  const int rc = check_4bit(n_kv_heads, head_dim, page_size);
  if (rc) return rc;
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(PKV_ERR_INVALID, "unsupported dtype code %d", dtype);
  if (n_rows < 0 || num_blocks < 0) return fail(PKV_ERR_INVALID, "negative count");
  if (n_rows == 0) return PKV_OK;
  if (!k_pool || !v_pool || !k || !v || !slots)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const FourBit f = four_bit(n_kv_heads, head_dim, page_size);
  hipStream_t s = (hipStream_t)stream;
  const int n = f.tiled ? 16 : 2;                  // elements of a thread
  if (((uintptr_t)k | (uintptr_t)v) % (std::min(n, 8) * eb))
    return fail(PKV_ERR_INVALID, "k and v have to be aligned to %d bytes", std::min(n, 8) * eb);
  const int per_head = head_dim / n, per_row = n_kv_heads * per_head;
  const int64_t total = n_rows > 0x7fffffffLL ? n_rows : n_rows * 2 * per_row;
  if (total > 0x7fffffffLL) return fail(PKV_ERR_INVALID, "too many rows in one read");
  auto go = [&](auto kernel, auto type) {
    typedef decltype(type) T;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, s,
                       (const unsigned char*)k_pool, (const unsigned char*)v_pool,
                       num_blocks * page_size, f, div_by(per_row), div_by(per_head),
                       div_by(page_size), slots, (uint32_t)total, (T*)k, (T*)v, status_word);
  };
  auto by_type = [&](auto type) {
    typedef decltype(type) T;
    if (f.tiled) go(read_4bit_kernel<T>, type);
    else go(read_4bit_any_kernel<T>, type);
  };
  if (dtype == PKV_DTYPE_F16) by_type(_Float16{});
  else if (dtype == PKV_DTYPE_BF16) by_type(__bf16{});
  else by_type(float{});
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

}  // extern "C"

namespace pkv {

// attend_4bit's geometries without a matrix-core kernel (arguments checked there)
int run_4bit_any(const pkv_4bit& b, const void* q, void* out, const void* k_pool,
                 const void* v_pool, float scale, hipStream_t s) {
  const FourBit f = four_bit(b.n_kv_heads, b.head_dim, b.page_size);
  const int64_t work = (int64_t)b.n_tokens * b.n_heads;
  if (!launchable(work, 64)) return fail(PKV_ERR_INVALID, "too many query rows");
  auto go = [&](auto type) {
    typedef decltype(type) T;
    hipLaunchKernelGGL(attend_4bit_any_kernel<T>, dim3((unsigned)work), dim3(64), 0, s,
                       (const T*)q, (T*)out, (const unsigned char*)k_pool,
                       (const unsigned char*)v_pool, b.num_blocks, f, b.cu_query_lens, b.kv_indptr,
                       b.kv_indices, b.kv_lens, b.batch_indices, b.n_seqs, b.n_heads,
                       scale * kLog2e, b.status_word);
  };
  if (b.dtype == PKV_DTYPE_F16) go(_Float16{});
  else if (b.dtype == PKV_DTYPE_BF16) go(__bf16{});
  else go(float{});
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

}  // namespace pkv
